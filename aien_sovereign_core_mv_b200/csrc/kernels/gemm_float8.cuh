// y[m][n] = sum over blocks b of 128 along K of (sum of a[m][k] w[n][k] over the block) * a_scales[b][m] * w_scales[n / 128][b], a and w
// e4m3 codes, on the fifth-generation tensor cores.  Part of gemm_tc.cu: the kernels share its error word.
//
// A row of a k-block of 128 codes is 128 bytes, one swizzled row of shared memory, so a k-block is what TMA brings, four
// instructions (K 32) multiply and one pair of scales belongs to.  The tensor cores add up one k-block at a time into one of several
// accumulators in tensor memory; the epilogue's warps read each of them, multiply by the scales and add to sums in
// registers, while the next k-blocks go into the other accumulators.  Everything that is added is float32.
//
// Two forms.  float8_few_kernel, for few rows of a: W's rows are the tensor memory's lanes (the M of the instruction) and the
// tokens its columns, so that a tile of W is 128 rows whatever the number of tokens; what bounds it is W's way through memory, so as many
// stages as fit are on their way, two CTAs on an SM, and a cluster of CTAs shares a tile's K where tiles are few.
// float8_tiles_kernel, for many: persistent, tokens are the lanes, tiles of 128 x BN; what bounds it is the tensor cores' rate.
// Rows and columns beyond the matrices are zero-filled by TMA, stores are masked.  Codes start on 16-byte borders, row by row.
#pragma once
#include "tma.cuh"
#include "umma.cuh"

namespace aien {

constexpr int F8_KB = 128;

// A matrix of codes [rows, cols], rows ld bytes apart, in boxes of box_rows rows x 128 codes, 128-byte swizzle, zeros beyond it.
inline bool f8_make_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {rows > 1 ? ld : (cols + 15) / 16 * 16};
    cuuint32_t box[2] = {(cuuint32_t)F8_KB, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct F8Scales {
    const float* a;       // [blocks][M], lda numbers apart
    long lda;
    const float* w;       // [ceil(N / 128)][blocks], ldw numbers apart
    long ldw;
};

// Two float32 numbers at a time: acc += v * s
__device__ __forceinline__ void f8_fma2(uint64_t& acc, uint32_t v0, uint32_t v1, uint64_t s) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s));
}
__device__ __forceinline__ uint64_t f8_two(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    return v;
}
__device__ __forceinline__ float2 f8_split(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ void f8_named_barrier(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

// ---------------------------------------------------------------- few rows of a
template <int NT> struct F8Few {
    static constexpr int STAGE_W = 128 * F8_KB, STAGE_A = NT * F8_KB;
    static constexpr int STAGES = NT == 16 ? 6 : NT == 32 ? 5 : 4;            // two CTAs on an SM: at most 113 KB each
    static constexpr int BUFS = 4, TMEM_COLS = BUFS * NT;                     // 64, 128 or 256 of 512 columns
    static constexpr int CHUNK = 32;                                          // k-blocks whose scales lie ready at a time
    static constexpr int FACTORS = CHUNK * NT * 4;
    static constexpr int SMEM = STAGES * (STAGE_W + STAGE_A) + FACTORS + 1024 /*align*/ + 256 /*barriers*/;
};

// blockIdx.x: the CTA's rank in the cluster (gridDim.x CTAs) that shares a tile's K; y: tile of NT tokens; z: tile of 128 rows of W.
template <int NT, typename TC>
__global__ void __launch_bounds__(192, 2)
float8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, F8Scales sc, TC* __restrict__ out, long ldc,
                  int M, int N, int K) {
    using C = F8Few<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sW = base, sA = base + C::STAGES * C::STAGE_W;
    float* factors = reinterpret_cast<float*>(gen + C::STAGES * (C::STAGE_W + C::STAGE_A));
    const uint32_t bars = base + C::STAGES * (C::STAGE_W + C::STAGE_A) + C::FACTORS;
    const uint32_t full0 = bars, empty0 = full0 + 8 * C::STAGES, tfull0 = empty0 + 8 * C::STAGES, tempty0 = tfull0 + 8 * C::BUFS, slot = tempty0 + 8 * C::BUFS;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + (slot - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x, Z = gridDim.x, m0 = blockIdx.y * NT, n0 = blockIdx.z * 128;
    const int total = (K + F8_KB - 1) / F8_KB;
    const int kb0 = (int)((long)total * rank / Z), num = (int)((long)total * (rank + 1) / Z) - kb0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < C::BUFS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"((uint32_t)C::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *slot_ptr;
    griddep_launch();                                                         // behind the allocation: what starts now cannot take these columns and wait for this kernel
    const int pt = threadIdx.x - 64;                                          // of the 128 threads that add up
    const int row = (warp & 3) * 32 + lane;                                   // the tensor memory's lane
    uint64_t acc[NT / 2];
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) acc[i] = 0;

    if (warp == 0) {
        if (lane == 0) {
            griddep_wait();
            for (int kb = 0; kb < num; ++kb) {
                const int s = kb % C::STAGES, round = kb / C::STAGES;
                if (round > 0) mbar_wait(empty0 + 8 * s, (round - 1) & 1, 1);
                mbar_expect_tx(full0 + 8 * s, C::STAGE_W + C::STAGE_A);
                tma_load_2d(sW + s * C::STAGE_W, &map_w, full0 + 8 * s, (kb0 + kb) * F8_KB, n0);
                tma_load_2d(sA + s * C::STAGE_A, &map_a, full0 + 8 * s, (kb0 + kb) * F8_KB, m0);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc_e4m3(128, NT);
            for (int kb = 0; kb < num; ++kb) {
                const int s = kb % C::STAGES, b = kb % C::BUFS, use = kb / C::BUFS;
                mbar_wait(full0 + 8 * s, (kb / C::STAGES) & 1, 2);
                if (use > 0) mbar_wait(tempty0 + 8 * b, (use - 1) & 1, 2);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t dw = make_desc_sw128(sW + s * C::STAGE_W), da = make_desc_sw128(sA + s * C::STAGE_A);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + b * NT, dw + 2 * k, da + 2 * k, idesc, k > 0 ? 1u : 0u);      // 32 codes = 2 descriptor units
                umma_commit(empty0 + 8 * s);
                umma_commit(tfull0 + 8 * b);
            }
        }
    } else {
        griddep_wait();
        for (int kb = 0; kb < num; ++kb) {
            if (kb % C::CHUNK == 0) {
                if (kb > 0) f8_named_barrier(128);                            // everyone is through with the scales before these
                const int count = min(C::CHUNK, num - kb) * NT;
                for (int i = pt; i < count; i += 128) {
                    const int b = kb0 + kb + i / NT, t = m0 + i % NT;
                    factors[i] = t < M ? __ldcg(sc.a + (long)b * sc.lda + t) * __ldcg(sc.w + (long)blockIdx.z * sc.ldw + b) : 0.f;
                }
                f8_named_barrier(128);
            }
            const int b = kb % C::BUFS;
            mbar_wait(tfull0 + 8 * b, (kb / C::BUFS) & 1, 3);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            __syncwarp();
            const ulonglong2* f = reinterpret_cast<const ulonglong2*>(factors + (kb % C::CHUNK) * NT);
#pragma unroll
            for (int c0 = 0; c0 < NT; c0 += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(b * NT + c0), r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const ulonglong2 s2 = f[c0 / 4 + j];
                    f8_fma2(acc[c0 / 2 + 2 * j], r[4 * j], r[4 * j + 1], s2.x);
                    f8_fma2(acc[c0 / 2 + 2 * j + 1], r[4 * j + 2], r[4 * j + 3], s2.y);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty0 + 8 * b);
        }
    }
    const int n = n0 + row;
    if (Z == 1) {
        if (warp >= 2 && n < N) {
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) {
                const float2 v = f8_split(acc[i]);
                if (m0 + 2 * i < M) out[(long)(m0 + 2 * i) * ldc + n] = from_f<TC>(v.x);
                if (m0 + 2 * i + 1 < M) out[(long)(m0 + 2 * i + 1) * ldc + n] = from_f<TC>(v.y);
            }
        }
    } else {
        // Every CTA of the cluster has its part of K behind it: the rings are free.  CTA z takes columns z * NT / Z .. of everyone's
        // sums ([rank][column][row] in its ring) and adds them up in the order of K.
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int cw = NT / Z;
        if (warp >= 2) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float2 v = f8_split(acc[c / 2]);
                const uint32_t to = tc_map_rank(base + (uint32_t)(((rank * cw + c % cw) * 128 + row) * 4), (uint32_t)(c / cw));
                asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(__float_as_uint(c & 1 ? v.y : v.x)) : "memory");
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp >= 2 && n < N) {
            const volatile float* part = reinterpret_cast<const volatile float*>(gen);
            for (int c = 0; c < cw && m0 + rank * cw + c < M; ++c) {
                float v = 0.f;
                for (int z = 0; z < Z; ++z) v += part[(z * cw + c) * 128 + row];
                out[(long)(m0 + rank * cw + c) * ldc + n] = from_f<TC>(v);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------- many rows of a
template <int BN> struct F8Tiles {
    static constexpr int STAGE_A = 128 * F8_KB, STAGE_W = BN * F8_KB;
    static constexpr int STAGES = 192 * 1024 / (STAGE_A + STAGE_W);           // 4 of 48 KB, 6 of 32 KB
    static constexpr int BUFS = 512 / BN;
    static constexpr int SMEM = STAGES * (STAGE_A + STAGE_W) + 1024 /*align*/ + 256 /*barriers*/;
};

// Warp 0 fetches, warp 1 multiplies, warps 2 to 9 add up: each a quarter of the tile's rows times half of its columns, a row a thread.
template <int BN, typename TC>
__global__ void __launch_bounds__(320, 1)
float8_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, F8Scales sc, TC* __restrict__ out, long ldc,
                    int M, int N, int K, int m_tiles, int tiles) {
    using C = F8Tiles<BN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sA = base, sW = base + C::STAGES * C::STAGE_A;
    const uint32_t bars = base + C::STAGES * (C::STAGE_W + C::STAGE_A);
    const uint32_t full0 = bars, empty0 = full0 + 8 * C::STAGES, tfull0 = empty0 + 8 * C::STAGES, tempty0 = tfull0 + 8 * C::BUFS, slot = tempty0 + 8 * C::BUFS;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + (slot - base));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (K + F8_KB - 1) / F8_KB;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < C::BUFS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *slot_ptr;
    griddep_launch();                                                         // behind the allocation: what starts now cannot take these columns and wait for this kernel

    if (warp == 0) {
        if (lane == 0) {
            griddep_wait();
            int it = 0;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                const int m0 = tile % m_tiles * 128, n0 = tile / m_tiles * BN;
                for (int kb = 0; kb < blocks; ++kb, ++it) {
                    const int s = it % C::STAGES, round = it / C::STAGES;
                    if (round > 0) mbar_wait(empty0 + 8 * s, (round - 1) & 1, 1);
                    mbar_expect_tx(full0 + 8 * s, C::STAGE_W + C::STAGE_A);
                    tma_load_2d(sA + s * C::STAGE_A, &map_a, full0 + 8 * s, kb * F8_KB, m0);
                    tma_load_2d(sW + s * C::STAGE_W, &map_w, full0 + 8 * s, kb * F8_KB, n0);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc_e4m3(128, BN);
            int it = 0;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                for (int kb = 0; kb < blocks; ++kb, ++it) {
                    const int s = it % C::STAGES, b = it % C::BUFS, use = it / C::BUFS;
                    mbar_wait(full0 + 8 * s, (it / C::STAGES) & 1, 2);
                    if (use > 0) mbar_wait(tempty0 + 8 * b, (use - 1) & 1, 2);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = make_desc_sw128(sA + s * C::STAGE_A), dw = make_desc_sw128(sW + s * C::STAGE_W);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_f8(tmem + b * BN, da + 2 * k, dw + 2 * k, idesc, k > 0 ? 1u : 0u);
                    umma_commit(empty0 + 8 * s);
                    umma_commit(tfull0 + 8 * b);
                }
            }
        }
    } else {
        griddep_wait();
        constexpr int W = BN / 2;                                             // a thread's columns
        const int quarter = warp & 3, c_first = (warp - 2) / 4 * W;
        // the factor of the k-block after the next one is on its way: (tile, k-block) runs ahead of the sums by two
        int ptile = blockIdx.x, pkb = 0;
        auto fetch = [&]() {
            float f = 0.f;
            if (ptile < tiles) {
                const int m = ptile % m_tiles * 128 + quarter * 32 + lane, n = ptile / m_tiles * BN + c_first;
                if (m < M && n < N) f = __ldcg(sc.a + (long)pkb * sc.lda + m) * __ldcg(sc.w + (long)(n / 128) * sc.ldw + pkb);
                if (++pkb == blocks) { pkb = 0; ptile += gridDim.x; }
            }
            return f;
        };
        float f1 = fetch(), f2 = fetch();
        int it = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            uint64_t acc[W / 2];
#pragma unroll
            for (int i = 0; i < W / 2; ++i) acc[i] = 0;
            for (int kb = 0; kb < blocks; ++kb, ++it) {
                const float f = f1;
                f1 = f2;
                f2 = fetch();
                const uint64_t s2 = f8_two(f, f);
                const int b = it % C::BUFS;
                mbar_wait(tfull0 + 8 * b, (it / C::BUFS) & 1, 3);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int c0 = 0; c0 < W; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * BN + c_first + c0), r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 16; ++j) f8_fma2(acc[c0 / 2 + j], r[2 * j], r[2 * j + 1], s2);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty0 + 8 * b);
            }
            const int m = tile % m_tiles * 128 + quarter * 32 + lane, n0 = tile / m_tiles * BN;
            if (m < M) {
#pragma unroll
                for (int c0 = 0; c0 < W; c0 += 32) {
                    uint32_t r[32];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 v = f8_split(acc[c0 / 2 + j]);
                        r[2 * j] = __float_as_uint(v.x);
                        r[2 * j + 1] = __float_as_uint(v.y);
                    }
                    if (n0 + c_first + c0 < N) tc_store_chunk<0, TC>(r, out, ldc, m, n0, c_first + c0, N);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---------------------------------------------------------------- host side
// The shared memory that a kernel needs, once for every device.
template <auto KERNEL, int SMEM>
inline bool f8_configure() {
    static std::once_flag once[64];
    static bool ok[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    std::call_once(once[dev], [&] { ok[dev] = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess; });
    return ok[dev];
}

template <typename... KArgs, typename... Args>
inline int f8_launch(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    return e != cudaSuccess ? (int)e : launch_status();
}

inline int f8_sms() {
    int sms = 148, dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    return sms;
}

template <int NT, typename TC>
int launch_float8_few(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, cudaStream_t stream) {
    CUtensorMap ma, mw;
    if (!f8_make_map(&ma, a, M, K, lda, NT) || !f8_make_map(&mw, w, N, K, ldw, 128)) return AIEN_E_STATE;
    auto kernel = float8_few_kernel<NT, TC>;
    if (!f8_configure<float8_few_kernel<NT, TC>, F8Few<NT>::SMEM>()) return AIEN_E_STATE;
    const long m_tiles = (M + NT - 1) / NT, n_tiles = (N + 127) / 128, blocks = (K + F8_KB - 1) / F8_KB;
    if (m_tiles > 65535 || n_tiles > 65535) return AIEN_E_SHAPE;
    int Z = 1;
    while (Z < 8 && Z * 2 <= blocks && m_tiles * n_tiles * Z * 2 <= 2 * f8_sms()) Z *= 2;
    return f8_launch(kernel, dim3(Z, (unsigned)m_tiles, (unsigned)n_tiles), 192, F8Few<NT>::SMEM, Z, stream, ma, mw, sc, (TC*)out, ldc, M, N, K);
}

template <int BN, typename TC>
int launch_float8_tiles(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, cudaStream_t stream) {
    CUtensorMap ma, mw;
    if (!f8_make_map(&ma, a, M, K, lda, 128) || !f8_make_map(&mw, w, N, K, ldw, BN)) return AIEN_E_STATE;
    auto kernel = float8_tiles_kernel<BN, TC>;
    if (!f8_configure<float8_tiles_kernel<BN, TC>, F8Tiles<BN>::SMEM>()) return AIEN_E_STATE;
    const long m_tiles = (M + 127) / 128, tiles = m_tiles * ((N + BN - 1) / BN);
    if (tiles * ((K + F8_KB - 1) / F8_KB) > 2147483647L) return AIEN_E_SHAPE;
    const int ctas = (int)(tiles < f8_sms() ? tiles : f8_sms());
    return f8_launch(kernel, dim3(ctas), 320, F8Tiles<BN>::SMEM, 1, stream, ma, mw, sc, (TC*)out, ldc, M, N, K, (int)m_tiles, (int)tiles);
}

template <typename TC>
int launch_float8(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, cudaStream_t stream) {
#define F8_FEW(NT) return launch_float8_few<NT, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, stream)
#define F8_TILES(BN) return launch_float8_tiles<BN, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, stream)
    if (M <= 16) F8_FEW(16);
    if (M <= 32) F8_FEW(32);
    if (M <= 256) F8_FEW(64);
    if (((long)(M + 127) / 128) * ((N + 255) / 256) >= f8_sms()) F8_TILES(256);
    F8_TILES(128);
#undef F8_FEW
#undef F8_TILES
}

}  // namespace aien

// Whether the tensor-core forms take codes that lie like this: every row on a 16-byte border.
AIEN_API int aien_matmul_float8_tc(const void* a, long lda, const float* sa, long lds, const void* w, long ldw, const float* sw, long ldsw,
                                   void* out, int c_dt, long ldc, int M, int N, int K, cudaStream_t stream) {
    using namespace aien;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return AIEN_E_SHAPE;
    if (((uintptr_t)a & 15) || ((uintptr_t)w & 15) || (M > 1 && (lda & 15)) || (N > 1 && (ldw & 15))) return AIEN_E_ALIGN;
    const F8Scales sc{sa, lds, sw, ldsw};
    AIEN_DISPATCH_DTYPE(c_dt, TC, return (launch_float8<TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, stream)));
}
