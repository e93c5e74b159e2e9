// Numbers in 8 bits (e4m3) with one float32 scale for each block of 128: rows (a norm's, a gated activation's, any) and weights
// in blocks of 128 x 128.
//
// A block with largest magnitude m gets the scale s = max(m * (1 / 448), 2^-126) and the codes e4m3(x * (1 / s)), to the nearest, ties to
// even, at most 448; both reciprocals and both products are rounded to float32.  A block of zeros has codes 0; a block that holds an infinity or something that is not a number has a
// scale and codes that are not numbers, so that a product's row shows it as the product of the unscaled row would.
// Largest magnitudes are taken over the bits of |x| as whole numbers: that order is the order of the numbers, and
// what is not a number comes out above infinity instead of being lost.
// Scales of rows are laid out [blocks, rows]: the products' kernels read a block's scales of neighbouring rows together.
//
// All of these are bound by memory, or for a few rows by latency: every number is read once, kept in registers while its block's
// (or row's) maximum is found, and written once.
#include "float8.cuh"

namespace aien {

// maximum over the 16 lanes that share a block
__device__ __forceinline__ uint32_t f8_half_max(uint32_t v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Eight numbers as they lie in memory, one or two 16-byte loads.  __ldcg: what an earlier kernel of a chain wrote (see common.cuh).
template <typename T> struct F8Raw;
template <> struct F8Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldcg(reinterpret_cast<const float4*>(p));
        b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void get(float v[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <> struct F8Raw<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldcg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void get(float v[8]) const {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <typename T>
__device__ __forceinline__ void f8_load8(const T* p, float v[8]) {
    F8Raw<T> r;
    r.load(p);
    r.get(v);
}

// ---------------------------------------------------------------- rows, and gated activations of rows
// Where the eight numbers of a lane come from.  Eight neighbours, loaded whole, where every row starts on a 16-byte border and holds whole eights (load and
// get); otherwise numbers lane, lane + 16, ... of the block, one by one (each).
template <typename T> struct F8Plain {
    static constexpr int CTAS = 8;                                             // on an SM: 32 registers a thread, 8,192 x 4,096 in 18.7 us for 19.6 with 40
    static constexpr float SIGN = 1.0f;
    const T* x;
    long ld;
    struct Raw { F8Raw<T> x; };
    __device__ __forceinline__ void load(long t, int i, int K, Raw& r) const { r.x.load(x + t * ld + i); }
    __device__ __forceinline__ void get(const Raw& r, float v[8]) const { r.x.get(v); }
    __device__ __forceinline__ float each(long t, int i, int K) const { return ld_act(x + t * ld + i); }
};
template <typename T, bool GELU> struct F8Gated {
    static constexpr int CTAS = sizeof(T) == 2 ? 6 : 4;                       // 40 or 64 registers; with 64 for bfloat16 too 2,048 x 12,288 in 28.2 us for 24.8
    static constexpr float SIGN = -1.0f;                                      // of the numbers that get and each give
    const T* gu;
    int group;
    struct Raw { F8Raw<T> g, u; };
    __device__ __forceinline__ void load(long t, int i, int K, Raw& r) const {
        const T* p = gu + t * 2 * (long)K;
        r.g.load(p + (group == 0 ? i : 2 * i));
        r.u.load(p + (group == 0 ? K + i : 2 * i + 8));
    }
    __device__ __forceinline__ void get(const Raw& r, float v[8]) const {
        float u[8];
        r.g.get(v);
        r.u.get(u);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 y = f8_split(f8_minus_gate<GELU>(f8_two(v[j], v[j + 1]), f8_two(u[j], u[j + 1])));
            v[j] = y.x;
            v[j + 1] = y.y;
        }
    }
    __device__ __forceinline__ float each(long t, int i, int K) const {
        const T* p = gu + t * 2 * (long)K;
        const long gi = group == 0 ? i : (long)(i / group) * 2 * group + i % group;
        return f8_minus_gate<GELU>(ld_act(p + gi), ld_act(p + gi + (group == 0 ? K : group)));
    }
};

template <bool VEC>
__device__ __forceinline__ void f8_store(uint8_t* codes, int k0, int lane, int K, const float v[8], float inv) {
    if (VEC) {
        *reinterpret_cast<uint2*>(codes + k0 + lane * 8) = f8_pack(v, inv);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = k0 + j * 16 + lane;
            if (k < K) codes[k] = (uint8_t)__nv_cvt_float_to_fp8(v[j] * inv, __NV_SATFINITE, __NV_E4M3);
        }
    }
}

// Half a warp takes a block of a row, U blocks of it one after the other whose loads are all on their way first.  A CTA's 16 halves are `rows` (2^rows_log2) rows times
// 16 / rows neighbouring blocks: one row where it has sixteen blocks, so that what a CTA reads lies together (gated, 512 x 12,288 in 8.3 us;
// two rows of eight 8.4, eight rows of two, whose scales leave together, 8.6).
// (As many CTAs as the GPU holds, walking over the blocks with the next one's numbers on their way, took longer: 2,048 x 12,288 gated in 37 us for 31.)
template <typename SRC, bool VEC, int U>
__global__ void __launch_bounds__(256, SRC::CTAS)
rows_float8_kernel(SRC src, uint8_t* codes, long ldq, float* scales, long lds, int T, int K, int rows_log2) {
    griddep_launch();
    griddep_wait();
    const int half = threadIdx.x >> 4, lane = threadIdx.x & 15, wide = 16 >> rows_log2;
    const long t = ((long)blockIdx.x << rows_log2) + (half & ((1 << rows_log2) - 1));
    const int b0 = blockIdx.y * wide * U + (half >> rows_log2);
    typename SRC::Raw raw[U];
    if (VEC) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (b0 + u * wide) * F8_BLOCK + lane * 8;
            if (t < T && i < K) src.load(t, i, K, raw[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int b = b0 + u * wide, k0 = b * F8_BLOCK;
        const bool mine = t < T && (VEC ? k0 + lane * 8 < K : k0 < K);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (mine) {
            if (VEC) {
                src.get(raw[u], v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + j * 16 + lane < K) v[j] = src.each(t, k0 + j * 16 + lane, K);
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, f8_bits(v[j]));
        top = f8_half_max(top);
        const float s = f8_scale(top), inv = SRC::SIGN * f8_inverse(s);
        if (mine) f8_store<VEC>(codes + t * ldq, k0, lane, K, v, inv);
        if (t < T && k0 < K && lane == 0) scales[(long)b * lds + t] = s;
    }
}

template <typename SRC, bool VEC, int U>
static int launch_rows_float8_by(SRC src, uint8_t* codes, long ldq, float* scales, long lds, int T, int K, cudaStream_t stream) {
    const int blocks = (K + F8_BLOCK - 1) / F8_BLOCK;
    int rows_log2 = 0;
    while (rows_log2 < 4 && 1 << rows_log2 < T && 16 >> rows_log2 > blocks) ++rows_log2;
    const int rows = 1 << rows_log2, each = 16 / rows * U;
    const long gx = ((long)T + rows - 1) / rows, gy = ((long)blocks + each - 1) / each;
    if (gy > 65535) return AIEN_E_SHAPE;
    launch_chain(rows_float8_kernel<SRC, VEC, U>, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, stream, src, codes, ldq, scales, lds, T, K, rows_log2);
    return launch_status();
}
// Two blocks a half from two loads of the GPU on (148 SMs of 128 halves): gated, 2,048 x 12,288 in 29.4 us by one and 25.0 by two, 512 x 12,288 in 8.7 and
// 8.3, but 64 x 12,288 in 2.5 and 3.0; rows of 2,048 x 4,096 in 6.5 and 6.2, of 512 x 4,096 in 2.5 and 2.9.
template <typename SRC>
static int launch_rows_float8(bool vec, SRC src, uint8_t* codes, long ldq, float* scales, long lds, int T, int K, cudaStream_t stream) {
    if (!vec) return launch_rows_float8_by<SRC, false, 1>(src, codes, ldq, scales, lds, T, K, stream);
    if ((long)T * ((K + F8_BLOCK - 1) / F8_BLOCK) >= 2L * 148 * 128) return launch_rows_float8_by<SRC, true, 2>(src, codes, ldq, scales, lds, T, K, stream);
    return launch_rows_float8_by<SRC, true, 1>(src, codes, ldq, scales, lds, T, K, stream);
}

// ---------------------------------------------------------------- the residual's sum and its norm
// x += sum of the parts; h = x / sqrt(mean x^2 + eps) * w; codes and scales of h.  One CTA a row, the row in registers (NV times eight
// numbers a thread) between the sum of squares and the codes; a block of 128 lies in half a warp.
template <typename TD, typename TW, int NV, int BS>
__global__ void __launch_bounds__(BS)
add_rmsnorm_float8_vec_kernel(float* x, const TD* delta, int nparts, size_t part_stride, const TW* w, float eps,
                              uint8_t* codes, long ldq, float* scales, long lds, int H) {
    __shared__ float red[32];
    griddep_launch();
    griddep_wait();
    const size_t base = (size_t)blockIdx.x * H;
    float v[NV][8];
    F8Raw<TW> wv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = (j * BS + threadIdx.x) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
        if (i < H) f8_load8(x + base + i, v[j]);
    }
    if (delta != nullptr) {
#pragma unroll 2
        for (int p = 0; p < nparts; ++p) {
            float d[NV][8];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = (j * BS + threadIdx.x) * 8;
                if (i < H) f8_load8(delta + (size_t)p * part_stride + base + i, d[j]);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if ((j * BS + threadIdx.x) * 8 < H) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[j][e] += d[j][e];
                }
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[j][e] * v[j][e];
        const int i = (j * BS + threadIdx.x) * 8;
        if (i >= H) continue;
        wv[j].load(w + i);                                                  // on its way while the sum is made
        if (delta != nullptr) {
            float4* o = reinterpret_cast<float4*>(x + base + i);
            o[0] = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
            o[1] = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
        }
    }
    const float rstd = 1.0f / sqrtf(block_sum(ss, red) / (float)H + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = (j * BS + threadIdx.x) * 8;
        uint32_t top = 0;
        if (i < H) {
            float g[8];
            wv[j].get(g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] = v[j][e] * rstd * g[e];
                top = max(top, f8_bits(v[j][e]));
            }
        }
        top = f8_half_max(top);
        const float s = f8_scale(top), inv = f8_inverse(s);
        if (i < H) {
            *reinterpret_cast<uint2*>(codes + (size_t)blockIdx.x * ldq + i) = f8_pack(v[j], inv);
            if ((threadIdx.x & 15) == 0) scales[(long)(i / F8_BLOCK) * lds + blockIdx.x] = s;
        }
    }
}

// Any row: the sum goes back to memory and is read again.
template <typename TD>
__global__ void __launch_bounds__(512)
add_rmsnorm_float8_kernel(float* x, const TD* delta, int nparts, size_t part_stride, const void* w, int wdt, float eps,
                          uint8_t* codes, long ldq, float* scales, long lds, int H) {
    __shared__ float red[32];
    griddep_launch();
    griddep_wait();
    const size_t base = (size_t)blockIdx.x * H;
    float ss = 0.f;
    for (int i = threadIdx.x; i < H; i += blockDim.x) {
        float v = x[base + i];
        if (delta != nullptr) {
            for (int p = 0; p < nparts; ++p) v += ld_act(delta + (size_t)p * part_stride + base + i);
            x[base + i] = v;
        }
        ss += v * v;
    }
    const float rstd = 1.0f / sqrtf(block_sum(ss, red) / (float)H + eps);       // (its barriers stand between the writes of x and the reads below)
    const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int blocks = (H + F8_BLOCK - 1) / F8_BLOCK;
    for (int b0 = 0; b0 < blocks; b0 += blockDim.x >> 4) {                       // every lane takes part in every round: the maximum is over whole halves
        const int b = b0 + half, k0 = b * F8_BLOCK;
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = k0 + j * 16 + lane;
            v[j] = k < H ? x[base + k] * rstd * ld_act_dyn(w, wdt, k) : 0.f;
            top = max(top, f8_bits(v[j]));
        }
        top = f8_half_max(top);
        const float s = f8_scale(top), inv = f8_inverse(s);
        f8_store<false>(codes + (size_t)blockIdx.x * ldq, k0, lane, H, v, inv);
        if (lane == 0 && b < blocks) scales[(long)b * lds + blockIdx.x] = s;
    }
}

template <typename TD>
static int launch_add_rmsnorm_float8(float* x, const TD* delta, int nparts, size_t part_stride, const void* w, int w_dt, float eps,
                                     uint8_t* codes, long ldq, float* scales, long lds, int T, int H, cudaStream_t stream) {
    const bool vec = H % 8 == 0 && part_stride % 8 == 0 && ldq % 8 == 0 && ((uintptr_t)codes & 7) == 0 &&
                     (((uintptr_t)x | (uintptr_t)delta | (uintptr_t)w) & 15) == 0;
#define F8_NORM_W(TW, NV, BS)                                                                                                               \
    launch_chain(add_rmsnorm_float8_vec_kernel<TD, TW, NV, BS>, dim3(T), dim3(BS), 0, stream, x, delta, nparts, part_stride, (const TW*)w, eps, \
                 codes, ldq, scales, lds, H)
#define F8_NORM(NV, BS)                              \
    do {                                             \
        if (w_dt == AIEN_DT_F32) F8_NORM_W(float, NV, BS); \
        else F8_NORM_W(__nv_bfloat16, NV, BS);       \
    } while (0)
    // Many rows of up to 4,096: sixteen numbers a thread, whose loads are more (512 rows in 6.5 us for 7.1, 8,192 in 59.3 for 62.0); few: eight (64 in 2.7 for 2.75).
    if (vec && H <= 8 * 256) F8_NORM(1, 256);
    else if (vec && H <= 16 * 256 && T >= 512) F8_NORM(2, 256);
    else if (vec && H <= 8 * 512) F8_NORM(1, 512);
    else if (vec && H <= 16 * 512) F8_NORM(2, 512);
    else if (vec && H <= 32 * 512) F8_NORM(4, 512);
    else
        launch_chain(add_rmsnorm_float8_kernel<TD>, dim3(T), dim3(512), 0, stream, x, delta, nparts, part_stride, w, w_dt, eps, codes, ldq, scales, lds, H);
#undef F8_NORM_W
#undef F8_NORM
    return launch_status();
}

// ---------------------------------------------------------------- weights
// A CTA takes a block of 128 x 128: 16 lanes a row of it, BS / 16 rows at a time, the whole block in registers until its maximum is known, as it lies in
// memory where it is loaded in eights (256 threads), number by number otherwise (1,024 threads, sixteen numbers each).
template <typename T, bool VEC, int BS>
__global__ void __launch_bounds__(BS)
blocks_float8_kernel(const T* w, long ldw, uint8_t* codes, long ldq, float* scales, long lds, int N, int K) {
    constexpr int PASSES = 2048 / BS;
    __shared__ uint32_t tops[32];
    const int n0 = blockIdx.y * F8_BLOCK + (threadIdx.x >> 4), k0 = blockIdx.x * F8_BLOCK, lane = threadIdx.x & 15;
    F8Raw<T> raw[VEC ? PASSES : 1];
    float v[VEC ? 1 : PASSES][8];
    auto mine = [&](int i) { return n0 + i * (BS / 16) < N && (!VEC || k0 + lane * 8 < K); };
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const T* p = w + (long)(n0 + i * (BS / 16)) * ldw + k0;
        if (VEC) {
            if (mine(i)) raw[i].load(p + lane * 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = mine(i) && k0 + j * 16 + lane < K ? ld_act(p + j * 16 + lane) : 0.f;
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        float (&u)[8] = v[VEC ? 0 : i];
        if (!mine(i)) continue;
        if (VEC) raw[i].get(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, f8_bits(u[j]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BS / 32; ++i) top = max(top, tops[i]);
    const float s = f8_scale(top), inv = f8_inverse(s);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        float (&u)[8] = v[VEC ? 0 : i];
        if (!mine(i)) continue;
        if (VEC) raw[i].get(u);
        f8_store<VEC>(codes + (long)(n0 + i * (BS / 16)) * ldq, k0, lane, K, u, inv);
    }
    if (threadIdx.x == 0) scales[(long)blockIdx.y * lds + blockIdx.x] = s;
}

}  // namespace aien

using namespace aien;

// x [T, K] rows of float32 or bfloat16 (ldx numbers apart) to codes [T, K] (ldq bytes apart) and scales [ceil(K / 128), T] (lds numbers apart)
AIEN_API int aien_quantize_rows_float8(const void* x, int dt, long ldx, void* codes, long ldq, float* scales, long lds, int T, int K, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (K <= 0) return AIEN_E_SHAPE;
    const bool ends = K % 8 == 0 && ldq % 8 == 0 && ((uintptr_t)codes & 7) == 0 && ((uintptr_t)x & 15) == 0;
#define F8_ROWS(TX, WHOLE) \
    return launch_rows_float8(ends && ldx % WHOLE == 0, F8Plain<TX>{(const TX*)x, ldx}, (uint8_t*)codes, ldq, scales, lds, T, K, stream)
    if (dt == AIEN_DT_F32) F8_ROWS(float, 4);
    if (dt == AIEN_DT_BF16) F8_ROWS(__nv_bfloat16, 8);
#undef F8_ROWS
    return AIEN_E_DTYPE;
}

// act(gate) * up of gate_up [T, 2K] (contiguous; group 0: gate columns first; else interleaved in runs of group), the same way
AIEN_API int aien_swiglu_float8(const void* gu, int dt, int group, int gelu, void* codes, long ldq, float* scales, long lds, int T, int K, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (K <= 0 || group < 0 || (group > 0 && K % group != 0)) return AIEN_E_SHAPE;
    const bool vec = K % 8 == 0 && ldq % 8 == 0 && ((uintptr_t)codes & 7) == 0 && ((uintptr_t)gu & 15) == 0 && (group == 0 || group == 8);
#define F8_GATED(TX)                                                                                                                                    \
    return gelu ? launch_rows_float8(vec, F8Gated<TX, true>{(const TX*)gu, group}, (uint8_t*)codes, ldq, scales, lds, T, K, stream)                     \
                : launch_rows_float8(vec, F8Gated<TX, false>{(const TX*)gu, group}, (uint8_t*)codes, ldq, scales, lds, T, K, stream)
    if (dt == AIEN_DT_F32) F8_GATED(float);
    if (dt == AIEN_DT_BF16) F8_GATED(__nv_bfloat16);
#undef F8_GATED
    return AIEN_E_DTYPE;
}

// delta: [nparts][T][H] (nparts >= 1; part_stride in numbers) or null
AIEN_API int aien_add_rmsnorm_float8(float* x, const void* delta, int delta_dt, int nparts, size_t part_stride, const void* w, int w_dt, float eps,
                                     void* codes, long ldq, float* scales, long lds, int T, int H, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (H <= 0 || (delta != nullptr && nparts < 1)) return AIEN_E_SHAPE;
    AIEN_DISPATCH_DTYPE(delta_dt, TD, return launch_add_rmsnorm_float8<TD>(x, (const TD*)delta, nparts, part_stride, w, w_dt, eps, (uint8_t*)codes, ldq,
                                                                           scales, lds, T, H, stream));
}

// w [N, K] (ldw numbers apart) to codes [N, K] and scales [ceil(N / 128), ceil(K / 128)]
AIEN_API int aien_quantize_blocks_float8(const void* w, int dt, long ldw, void* codes, long ldq, float* scales, long lds, int N, int K, cudaStream_t stream) {
    if (N <= 0) return 0;
    if (K <= 0) return AIEN_E_SHAPE;
    const long gy = ((long)N + F8_BLOCK - 1) / F8_BLOCK;
    if (gy > 65535) return AIEN_E_SHAPE;
    const dim3 grid((K + F8_BLOCK - 1) / F8_BLOCK, (unsigned)gy);
    const bool ends = K % 8 == 0 && ldq % 8 == 0 && ((uintptr_t)codes & 7) == 0 && ((uintptr_t)w & 15) == 0;
#define F8_BLOCKS(TX, WHOLE)                                                                                                        \
    do {                                                                                                                            \
        if (ends && ldw % WHOLE == 0) blocks_float8_kernel<TX, true, 256><<<grid, 256, 0, stream>>>((const TX*)w, ldw, (uint8_t*)codes, ldq, scales, lds, N, K); \
        else blocks_float8_kernel<TX, false, 1024><<<grid, 1024, 0, stream>>>((const TX*)w, ldw, (uint8_t*)codes, ldq, scales, lds, N, K); \
        return launch_status();                                                                                                     \
    } while (0)
    if (dt == AIEN_DT_F32) F8_BLOCKS(float, 4);
    if (dt == AIEN_DT_BF16) F8_BLOCKS(__nv_bfloat16, 8);
#undef F8_BLOCKS
    return AIEN_E_DTYPE;
}
