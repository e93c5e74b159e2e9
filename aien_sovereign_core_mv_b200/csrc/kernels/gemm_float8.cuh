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
// float8_tiles_kernel, for many: persistent, tokens are the lanes, tiles of 128 x 128, or 256 x 256 by a pair of CTAs; what bounds it is the tensor cores' rate.
// Rows and columns beyond the matrices are zero-filled by TMA, stores are masked.  Rows of codes that do not all start on 16-byte borders
// are brought by threads in TMA's place (f8_gather).
#pragma once
#include "float8.cuh"
#include "tma.cuh"
#include "umma.cuh"
#include <atomic>

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

// The result [rows, cols], ld numbers between rows, in boxes of 32 rows x 128 bytes that a warp stores.
template <typename TC>
inline bool f8_make_map_out(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {rows > 1 ? ld * sizeof(TC) : (cols * sizeof(TC) + 15) / 16 * 16};
    cuuint32_t box[2] = {(cuuint32_t)(128 / sizeof(TC)), 32};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, sizeof(TC) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
__device__ __forceinline__ void f8_named_barrier(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }

__device__ __forceinline__ float4 f8_lds4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// lane 0 arrives, without a branch
__device__ __forceinline__ void f8_arrive0(uint32_t bar, int lane) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"(lane) : "memory");
}
__device__ __forceinline__ void f8_arrive0_cluster(uint32_t bar, int lane) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar), "r"(lane) : "memory");
}

// A place in a ring of N and the parity of the round that it is in.
template <int N> struct F8Ring {
    uint32_t at = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) { at = 0; parity ^= 1; }
    }
};

// Waits until the last rounds of a ring of stages have been multiplied: every arrival at its barriers is then behind, and the CTA may leave.  A stage that
// was never used passes at once, as it does in its first round.
template <int N>
__device__ __forceinline__ void f8_drain(uint32_t empty0, F8Ring<N> r) {
    for (int i = 0; i < N; ++i, r.next()) mbar_wait(empty0 + 8 * r.at, r.parity ^ 1, 1);
}

__device__ __forceinline__ bool f8_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// mbar_wait for a barrier that the other CTA of a pair arrives at too
__device__ __forceinline__ void f8_wait_cluster(uint32_t bar, uint32_t parity, int code) {
    for (uint32_t i = 0; i < TC_SPIN_LIMIT; ++i) {
        if (f8_try_wait_cluster(bar, parity)) return;
        if ((i & 0xFFFFFu) == 0xFFFFFu && *reinterpret_cast<volatile int*>(&g_wait_error) != 0) return;
    }
    atomicCAS(&g_wait_error, 0, code);
}

// All loads of tensor memory so far are in r.  (r goes through the wait: what is made of it in registers alone, which no order of volatile statements holds
// back, cannot be moved ahead of it.)
__device__ __forceinline__ void f8_tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
__device__ __forceinline__ void f8_tmem_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
    asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
                   "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}

// bytes of this CTA's shared memory to another one's of the cluster, which counts at a barrier there
__device__ __forceinline__ void f8_copy_to_rank(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}

// ---------------------------------------------------------------- few rows of a
template <int NT> struct F8Few {
    static constexpr int STAGE_W = 128 * F8_KB, STAGE_A = NT * F8_KB;
    static constexpr int STAGES = NT == 64 ? 3 : NT == 32 ? 4 : 5;            // two CTAs on an SM: at most 113 KB each
    static constexpr int PARTS = NT * 128 * 4;                                // what the CTAs of a cluster send each other
    static constexpr int BUFS = 4, TMEM_COLS = BUFS * NT;                     // 64, 128 or 256 of 512 columns
    static constexpr int CHUNK = NT == 64 ? 16 : 32;                          // k-blocks whose scales lie ready at a time
    static constexpr int FACTORS = CHUNK * NT * 4;
    static constexpr int SMEM = STAGES * (STAGE_W + STAGE_A) + PARTS + FACTORS + 1024 /*align*/ + 256 /*barriers*/;
};

// blockIdx.x: the CTA's rank in the cluster (gridDim.x CTAs) that shares a tile's K; y: tile of NT tokens; z: tile of 128 rows of W.
template <int NT, typename TC>
__global__ void __launch_bounds__(192, 2)
float8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, F8Scales sc, TC* __restrict__ out, long ldc,
                  int M, int N, int K, int w_ready) {
    using C = F8Few<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sW = base, sA = base + C::STAGES * C::STAGE_W;
    const uint32_t sParts = base + C::STAGES * (C::STAGE_W + C::STAGE_A);
    float* factors = reinterpret_cast<float*>(gen + C::STAGES * (C::STAGE_W + C::STAGE_A) + C::PARTS);
    const uint32_t bars = sParts + C::PARTS + C::FACTORS;
    const uint32_t full0 = bars, empty0 = full0 + 8 * C::STAGES, tfull0 = empty0 + 8 * C::STAGES, tempty0 = tfull0 + 8 * C::BUFS, parts_in = tempty0 + 8 * C::BUFS,
                   slot = parts_in + 8;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + (slot - base));
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;       // (known to be the same for the whole warp)
    const int rank = blockIdx.x, Z = gridDim.x, m0 = blockIdx.y * NT, n0 = blockIdx.z * 128;
    const int total = (K + F8_KB - 1) / F8_KB;
    const int kb0 = (int)((long)total * rank / Z), num = (int)((long)total * (rank + 1) / Z) - kb0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < C::BUFS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 4); }
        mbar_init(parts_in, 1);
        if (Z > 1) mbar_expect_tx(parts_in, (Z - 1) * (C::PARTS / Z));
        prefetch_map(&map_w);
        prefetch_map(&map_a);
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
    if (Z > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");          // this CTA runs and its barriers are there
    const int pt = threadIdx.x - 64;                                          // of the 128 threads that add up
    const int row = (warp & 3) * 32 + lane;                                   // the tensor memory's lane
    uint64_t acc[NT / 2];
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) acc[i] = 0;

    if (warp == 0) {
        // W's first stages are requested ahead of the wait for the kernel before this one where the caller says that W was there before it
        const int ahead = w_ready ? min(num, C::STAGES) : 0;
        if (elect_one()) {
            for (int kb = 0; kb < ahead; ++kb) {
                mbar_expect_tx(full0 + 8 * kb, C::STAGE_W + C::STAGE_A);
                tma_load_2d(sW + kb * C::STAGE_W, &map_w, full0 + 8 * kb, (kb0 + kb) * F8_KB, n0);
            }
        }
        __syncwarp();
        griddep_wait();
        F8Ring<C::STAGES> r;
        for (int kb = 0; kb < num; ++kb, r.next()) {
            mbar_wait(empty0 + 8 * r.at, r.parity ^ 1, 1);                    // (passes at once in the first round)
            if (elect_one()) {
                if (kb >= ahead) {
                    mbar_expect_tx(full0 + 8 * r.at, C::STAGE_W + C::STAGE_A);
                    tma_load_2d(sW + r.at * C::STAGE_W, &map_w, full0 + 8 * r.at, (kb0 + kb) * F8_KB, n0);
                }
                tma_load_2d(sA + r.at * C::STAGE_A, &map_a, full0 + 8 * r.at, (kb0 + kb) * F8_KB, m0);
            }
            __syncwarp();
        }
        f8_drain(empty0, r);
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_e4m3(128, NT);
        const uint64_t dw0 = make_desc_sw128(sW), da0 = make_desc_sw128(sA);
        F8Ring<C::STAGES> r;
        F8Ring<C::BUFS> t;
        for (int kb = 0; kb < num; ++kb, r.next(), t.next()) {
            const uint64_t dw = dw0 + r.at * (C::STAGE_W >> 4), da = da0 + r.at * (C::STAGE_A >> 4);
            mbar_wait(full0 + 8 * r.at, r.parity, 2);
            mbar_wait(tempty0 + 8 * t.at, t.parity ^ 1, 2);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + t.at * NT, dw + 2 * k, da + 2 * k, idesc, k > 0 ? 1u : 0u);        // 32 codes = 2 descriptor units
                umma_commit(tfull0 + 8 * t.at);
                umma_commit(empty0 + 8 * r.at);
            }
            __syncwarp();
        }
    } else {
        griddep_wait();
        F8Ring<C::BUFS> t;
        for (int kb = 0; kb < num; ++kb, t.next()) {
            if (kb % C::CHUNK == 0) {
                if (kb > 0) f8_named_barrier(128);                            // everyone is through with the scales before these
                const int count = min(C::CHUNK, num - kb) * NT;
                for (int i = pt; i < count; i += 128) {
                    const int b = kb0 + kb + i / NT, m = m0 + i % NT;
                    factors[i] = m < M ? __ldcg(sc.a + (long)b * sc.lda + m) * __ldcg(sc.w + (long)blockIdx.z * sc.ldw + b) : 0.f;
                }
                f8_named_barrier(128);
            }
            mbar_wait(tfull0 + 8 * t.at, t.parity, 3);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            __syncwarp();                                                     // (the loads of tensor memory are the whole warp's)
            const ulonglong2* f = reinterpret_cast<const ulonglong2*>(factors + (kb % C::CHUNK) * NT);
#pragma unroll
            for (int c0 = 0; c0 < NT; c0 += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(t.at * NT + c0), r);
                f8_tmem_wait(r);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const ulonglong2 s2 = f[c0 / 4 + j];
                    f8_fma2(acc[c0 / 2 + 2 * j], r[4 * j], r[4 * j + 1], s2.x);
                    f8_fma2(acc[c0 / 2 + 2 * j + 1], r[4 * j + 2], r[4 * j + 3], s2.y);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            f8_arrive0(tempty0 + 8 * t.at, lane);
        }
    }
    if (Z == 1) {                                                             // nobody to add to: straight from the registers
        const int n = n0 + row;
        if (warp >= 2 && n < N) {
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) {
                const float2 v = f8_split(acc[i]);
                if (m0 + 2 * i < M) out[(long)(m0 + 2 * i) * ldc + n] = from_f<TC>(v.x);
                if (m0 + 2 * i + 1 < M) out[(long)(m0 + 2 * i + 1) * ldc + n] = from_f<TC>(v.y);
            }
        }
    } else {
        // The sums go into the ring, whose last stage has been multiplied, [column][row].  CTA z takes columns z * NT / Z .. of everyone's: one
        // copy a CTA brings them to [from][column][row] in the owner's place for them (stored over the cluster number by number they took 2 us).
        const int cw = NT / Z;
        const uint32_t piece = C::PARTS / Z;
        if (warp >= 2) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float2 v = f8_split(acc[c / 2]);
                reinterpret_cast<float*>(gen)[c * 128 + row] = c & 1 ? v.y : v.x;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            f8_named_barrier(128);
        }
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // everyone runs
        if (warp == 2 && elect_one()) {
            for (int z = 0; z < Z; ++z)
                if (z != rank) f8_copy_to_rank(tc_map_rank(sParts + rank * piece, z), base + z * piece, piece, tc_map_rank(parts_in, z));
        }
        __syncwarp();
        if (warp >= 2) f8_wait_cluster(parts_in, 0, 3);
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // what others sent has arrived: when everyone says so, everyone may leave
        if (warp >= 2) {
            // Added up in the order of K.  Where two numbers make an aligned word, a thread takes two neighbours of every other column (one number of
            // every column: 64 x 4,096 x 12,288 in 17.3 us for 16.2).
            const bool two = (((uintptr_t)out | (uintptr_t)ldc * sizeof(TC)) & (2 * sizeof(TC) - 1)) == 0;
            const int r = two ? 2 * (pt & 63) : pt, n = n0 + r, step = two ? 2 : 1;
#pragma unroll 2
            for (int c = two ? pt >> 6 : 0; c < cw; c += step) {
                const int m = m0 + rank * cw + c;
                float2 v = make_float2(0.f, 0.f);
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    if (z >= Z) break;
                    const float* p = reinterpret_cast<const float*>((z == rank ? gen : gen + (sParts - base)) + z * piece) + c * 128 + r;
                    if (two) {
                        const float2 q = *reinterpret_cast<const float2*>(p);
                        v.x += q.x;
                        v.y += q.y;
                    } else {
                        v.x += *p;
                    }
                }
                if (m >= M || n >= N) continue;
                TC* to = out + (long)m * ldc + n;
                if (two && n + 1 < N) {
                    if constexpr (sizeof(TC) == 2) *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(v.x, v.y);
                    else *reinterpret_cast<float2*>(to) = v;
                } else {
                    *to = from_f<TC>(v.x);
                }
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------- many rows of a
// The scales' way: a warp copies those of four k-blocks at a time, of the tile's rows ([row][4]) and of its blocks of W ([2][4]), into a ring of
// slots ahead of the sums (a load that a warp of the sums waits for, even one issued two k-blocks before, cost a third of the kernel's time).
constexpr int F8_BATCH = 4, F8_SLOTS = 3, F8_SLOT = 130 * F8_BATCH * 4;
__device__ __forceinline__ void f8_copy4(uint32_t dst, const float* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4u : 0u) : "memory");
}
// k-blocks b .. b + 3: rows m0 .., blocks of W from nb on
__device__ __forceinline__ void f8_copy_scales(uint32_t dst, uint32_t bar, const F8Scales& sc, int b, int blocks, int m0, int M, int nb, int n_blocks, int lane) {
#pragma unroll
    for (int k = 0; k < F8_BATCH; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + i * 32 + lane;
            const bool live = m < M && b + k < blocks;
            f8_copy4(dst + ((i * 32 + lane) * F8_BATCH + k) * 4, live ? sc.a + (long)(b + k) * sc.lda + m : sc.a, live);
        }
    if (lane < 2 * F8_BATCH) {
        const int n = nb + lane / F8_BATCH, k = b + lane % F8_BATCH;
        const bool live = n < n_blocks && k < blocks;
        f8_copy4(dst + (128 * F8_BATCH + lane) * 4, live ? sc.w + (long)n * sc.ldw + k : sc.w, live);
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// acc += (W columns of a k-block's sums at taddr) * f; the next 32 columns are on their way while 32 are added.  read(): called when the last of
// them has left tensor memory.
template <int W, typename Read>
__device__ __forceinline__ void f8_add_block(uint32_t taddr, float f, float (&acc)[W], Read read) {
    static_assert(W % 64 == 0, "two registers' worth at a time");
    uint32_t r0[32], r1[32];
    tmem_ld32(taddr, r0);
#pragma unroll
    for (int c0 = 0; c0 < W; c0 += 64) {
        f8_tmem_wait(r0);
        tmem_ld32(taddr + c0 + 32, r1);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[c0 + j] = fmaf(__uint_as_float(r0[j]), f, acc[c0 + j]);
        f8_tmem_wait(r1);
        if (c0 + 64 < W) tmem_ld32(taddr + c0 + 64, r0);
        else read();
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[c0 + 32 + j] = fmaf(__uint_as_float(r1[j]), f, acc[c0 + 32 + j]);
    }
}

// A warp's 32 rows x W columns of the result, a row a lane.  By TMA (the result's rows start on 16-byte borders): 128 bytes of a row at a time into
// a buffer of 4 KB, 16-byte pieces swizzled as the copy expects them; rows and columns beyond the matrix are clipped by it.
// Other results leave the buffer row after row.  Stored from registers each lane's 16 bytes are a row of their own (a tile of 128 x 256 took 6,700 cycles so).
constexpr int F8_STORE = 4096;
template <int W, typename TC>
__device__ __forceinline__ void f8_store_rows(const float (&acc)[W], const CUtensorMap* map, bool by_tma, uint32_t at, TC* out, long ldc, int m, int n, int M, int N) {
    const int lane = threadIdx.x & 31;
    constexpr int COLS = 128 / sizeof(TC);
#pragma unroll
    for (int c0 = 0; c0 < W; c0 += COLS) {
        // (a copy writes whole 16-byte words: a box in which rows end inside one would take what lies behind them along)
        const bool leaves = by_tma && (n + c0 + COLS <= N || N % (16 / (int)sizeof(TC)) == 0);
        if (by_tma && lane == 0) tma_store_read<0>();                         // the last copy has read the buffer
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            uint4 v;
            if (sizeof(TC) == 2) {
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(acc[c0 + p * 8 + 2 * i], acc[c0 + p * 8 + 2 * i + 1]);
                    h[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
                v = make_uint4(h[0], h[1], h[2], h[3]);
            } else {
                v = make_uint4(__float_as_uint(acc[c0 + p * 4]), __float_as_uint(acc[c0 + p * 4 + 1]), __float_as_uint(acc[c0 + p * 4 + 2]), __float_as_uint(acc[c0 + p * 4 + 3]));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 128 + ((p ^ (lane & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        if (leaves) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (m < M && n + c0 < N) tma_store_2d(at, map, n + c0, m);
                tma_store_commit();
            }
        } else {                                                              // row after row, neighbouring lanes neighbouring numbers
            __syncwarp();
            const int end = n + c0 < N ? min(32, M - m) : 0;
#pragma unroll 4
            for (int r = 0; r < end; ++r) {
                TC* to = out + (long)(m + r) * ldc + n + c0;
#pragma unroll
                for (int c = lane; c < COLS; c += 32) {
                    const uint32_t from = at + r * 128 + ((((uint32_t)c * (uint32_t)sizeof(TC)) >> 4 ^ (r & 7)) << 4) + (c * sizeof(TC) & 15);
                    TC v;
                    if constexpr (sizeof(TC) == 2) {
                        uint16_t h;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from) : "memory");
                        v = __ushort_as_bfloat16(h);
                    } else {
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
                    }
                    if (n + c0 + c < N) to[c] = v;
                }
            }
            __syncwarp();
        }
    }
}

// PAIR: two CTAs make a tile of 256 x 256 together (cta_group::2): each holds 128 rows of a and half of the tile's rows of W in its shared memory,
// and the sums of its own rows in its tensor memory; the first issues the instructions for both.  Alone, a CTA makes 128 x 128.
// Shared memory is what the tensor cores wait for next: per k-block of 128 x 256 sums an SM's take 64 KB out of it in a pair and 96 alone, 128 as two
// of 128 x 128, beside the 32, 48 or 64 that TMA puts in, at 128 bytes a cycle, while the sums take 512 cycles.
constexpr int F8_RAW_ROW = 144, F8_RAW = 256 * F8_RAW_ROW, F8_RAWS = 3;                   // rows as they lie in memory: a k-block's, so many of them
// GATHER: the ring is two stages, the rest of its room the rows as they lie in memory.
template <bool PAIR, bool GATHER> struct F8Tiles {
    static constexpr int P = PAIR ? 2 : 1, BM = 128 * P, BN = 128 * P;
    static constexpr int STAGE_A = 128 * F8_KB, STAGE_W = 128 * F8_KB, STAGES = GATHER ? 2 : 5;
    static constexpr int BUFS = 512 / BN;
    static constexpr int RING = STAGES * (STAGE_A + STAGE_W), STORES = 8 * F8_STORE, RAWS = GATHER ? F8_RAWS * F8_RAW : 0;
    static constexpr int SMEM = RING + RAWS + STORES + F8_SLOTS * F8_SLOT + 1024 /*align*/ + 256 /*barriers*/;
    static_assert(SMEM <= 227 * 1024, "a CTA's shared memory");
};

// Rows of codes that start anywhere, which TMA does not take: 128 threads bring a k-block of a tile's 128 + 128 rows.  First as it lies in memory, in the nine
// 16-byte words that the 128 codes of a row touch, asynchronously and two k-blocks ahead; then shifted into place, where TMA would have put it.  Codes
// beyond a row and rows beyond the matrix become zeros.  Nothing outside the matrix is read: the copy of a word stops at its row's end, and the
// one word that may begin before the matrix is put together from its bytes.
struct F8Rows {
    const uint8_t* a;
    long lda;
    const uint8_t* w;
    long ldw;
};
// What a thread copies of a tile: word 16 * (thread + 128 i) of the k-block's 256 rows of nine, from its place in the first k-block on; how many codes of its row
// lie behind its beginning.
struct F8Words {
    const uint8_t* word[18];
    int left[18];
    __device__ __forceinline__ void start(const F8Rows& t, int m0, int M, int n0, int N, int K, int thread) {
        int row = thread / 9, c = thread % 9;
#pragma unroll
        for (int i = 0; i < 18; ++i) {
            const int r = row < 128 ? m0 + row : n0 + row - 128;
            const bool live = r < (row < 128 ? M : N);
            const uint8_t* begin = row < 128 ? t.a + (live ? (long)r * t.lda : 0) : t.w + (live ? (long)r * t.ldw : 0);
            const uint32_t off = (uint32_t)(uintptr_t)begin & 15;
            word[i] = begin - off + 16 * c;
            left[i] = !live || (c == 8 && off == 0) ? -1 : (int)off + K - 16 * c;           // (the ninth word of a row that starts on a border is the next k-block's)
            if (live) left[i] = max(left[i], -1);
            row += 14;                                                        // 128 = 14 x 9 + 2
            c += 2;
            if (c >= 9) { c -= 9; ++row; }
        }
    }
    // k-block kb's into the raw rows at `raw`
    __device__ __forceinline__ void copy(uint32_t raw, const F8Rows& t, int kb, int thread) const {
#pragma unroll
        for (int i = 0; i < 18; ++i) {
            const uint8_t* from = word[i] + (long)kb * F8_KB;
            const int bytes = min(max(left[i] - kb * F8_KB, 0), 16);
            const uint32_t dst = raw + 16 * (thread + 128 * i);
            if ((i == 0 || i == 9) && from < (i == 0 ? t.a : t.w) && bytes > 0) {           // thread 0, the matrix' first word: it begins before the matrix
                uint32_t v[4] = {0, 0, 0, 0};
                for (int b = 0; b < 16; ++b)
                    if (from + b >= (i == 0 ? t.a : t.w) && b < bytes) v[b >> 2] |= (uint32_t)__ldcg(from + b) << (8 * (b & 3));
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
            } else {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(bytes > 0 ? from : word[i]), "r"(bytes) : "memory");
            }
        }
    }
};
// How far a thread's sixteen rows ((thread / 8) + 16 i of the tile's 256) start behind a border, four bits each.
__device__ __forceinline__ uint64_t f8_offsets(const F8Rows& t, int m0, int n0, int thread) {
    uint64_t packed = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = (thread >> 3) + i * 16;
        const uint8_t* p = row < 128 ? t.a + (long)(m0 + row) * t.lda : t.w + (long)(n0 + row - 128) * t.ldw;
        packed |= (uint64_t)((uintptr_t)p & 15) << (4 * i);
    }
    return packed;
}
// 16 codes of each of those rows, chunk thread % 8, from the raw rows to where TMA would have put them
__device__ __forceinline__ void f8_place_raw(uint32_t raw, uint32_t tile_a, uint32_t tile_w, uint64_t offsets, int thread) {
    const int chunk = thread & 7, first = thread >> 3;
    const uint32_t from = raw + first * F8_RAW_ROW + chunk * 16, to = first * 128 + ((chunk ^ (first & 7)) << 4);
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const uint32_t s = (uint32_t)(offsets >> (4 * i)) & 15, at = from + i * (16 * F8_RAW_ROW);
        uint32_t v[8];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(at + 16) : "memory");
#pragma unroll
        for (int j = 0; j < 6; ++j) v[j] = s & 8 ? v[j + 2] : v[j];
#pragma unroll
        for (int j = 0; j < 5; ++j) v[j] = s & 4 ? v[j + 1] : v[j];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __funnelshift_r(v[j], v[j + 1], (s & 3) * 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((i < 8 ? tile_a + to + i * 2048 : tile_w + to + (i - 8) * 2048)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                     "r"(v[3]) : "memory");
    }
}

// Where a gated product's result goes: codes [M, N / 2] and scales [ceil(N / 256), M].
struct F8Gated8 {
    uint8_t* codes;
    long ldq;
    float* scales;
    long lds;
    int gelu;
};
// act(gate) * up of 128 columns in runs of 8, in the first 64 of them; their largest
template <bool GELU>
__device__ __forceinline__ uint32_t f8_gate_columns(float (&acc)[128], int n, int N) {
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < 8; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = -f8_minus_gate<GELU>(acc[16 * v + j], acc[16 * v + 8 + j]);
            acc[8 * v + j] = y;
            if (n + 16 * v < N) top = max(top, f8_bits(y));
        }
    return top;
}
// act(gate) * up of a row's 128 columns, which hold gate and up in runs of 8, in 8 bits.  A tile's 256 columns give the 128 numbers of one block: the two
// threads of a row tell each other their largest (`tops`, two floats a row).  All of it is float32: the columns are never rounded to 16 bits.
__device__ __forceinline__ void f8_store_gated(float (&acc)[128], const F8Gated8& g, uint32_t tops, int half, int row, int m, int n, int M, int N) {
    const uint32_t top = g.gelu ? f8_gate_columns<true>(acc, n, N) : f8_gate_columns<false>(acc, n, N);
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(tops + (half * 128 + row) * 4), "r"(top) : "memory");
    asm volatile("bar.sync 2, 256;" ::: "memory");
    uint32_t other;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(other) : "r"(tops + ((half ^ 1) * 128 + row) * 4) : "memory");
    const float s = f8_scale(max(top, other)), inv = f8_inverse(s);
    if (m >= M) return;
    if (half == 0) g.scales[(long)(n / 256) * g.lds + m] = s;
    uint8_t* to = g.codes + (long)m * g.ldq + n / 2;
    const bool whole = ((uintptr_t)to & 7) == 0;
#pragma unroll
    for (int v = 0; v < 8; ++v) {
        if (n + 16 * v >= N) continue;
        const uint2 c = f8_pack(&acc[8 * v], inv);
        if (whole) {
            *reinterpret_cast<uint2*>(to + 8 * v) = c;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) to[8 * v + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
        }
    }
}

// Persistent.  Warp 0 fetches, warp 1 multiplies, warp 2 brings the scales, warps 4 to 11 add up: each a quarter of the tile's rows times half
// of its columns, a row a thread; they take the registers that the first four give up.  GATHER: four more warps fetch in warp 0's place.
// GATED (in pairs): W's rows are gate and up in runs of 8, the result is act(gate) * up in 8 bits.
template <bool PAIR, bool GATHER, bool GATED, typename TC>
__global__ void __launch_bounds__(GATHER ? 512 : 384, 1)
float8_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
                    int store_by_tma, F8Scales sc, TC* __restrict__ out, long ldc, int M, int N, int K, int m_tiles, int tiles, F8Rows rows, F8Gated8 gated) {
    static_assert(!(PAIR && GATHER), "rows that start anywhere are multiplied in tiles of one CTA");
    static_assert(PAIR || !GATED, "a block of a gated result is 256 columns");
    using C = F8Tiles<PAIR, GATHER>;
    constexpr int P = C::P;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sA = base, sW = base + C::STAGES * C::STAGE_A, sRaw = base + C::RING, sStore = sRaw + C::RAWS, sScale = sStore + C::STORES;
    const uint32_t bars = sScale + F8_SLOTS * F8_SLOT;
    const uint32_t full0 = bars, empty0 = full0 + 8 * C::STAGES, tfull0 = empty0 + 8 * C::STAGES, tempty0 = tfull0 + 8 * C::BUFS;
    const uint32_t sfull0 = tempty0 + 8 * C::BUFS, sempty0 = sfull0 + 8 * F8_SLOTS, slot = sempty0 + 8 * F8_SLOTS;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(gen + (slot - base));
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;       // (known to be the same for the whole warp)
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0, first = (int)blockIdx.x / P, step = (int)gridDim.x / P;
    const int blocks = (K + F8_KB - 1) / F8_KB;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full0 + 8 * s, GATHER ? 128 : 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < C::BUFS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 8 * P); }
        for (int s = 0; s < F8_SLOTS; ++s) { mbar_init(sfull0 + 8 * s, 32); mbar_init(sempty0 + 8 * s, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) {                                                               // both have their barriers and their columns
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *slot_ptr;
    griddep_launch();                                                         // behind the allocation: what starts now cannot take these columns and wait for this kernel

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && !GATHER) {
            griddep_wait();
            F8Ring<C::STAGES> r;
            for (int tile = first; tile < tiles; tile += step) {
                const int m0 = tile % m_tiles * C::BM + rank * 128, n0 = tile / m_tiles * C::BN + rank * 128;
                for (int kb = 0; kb < blocks; ++kb, r.next()) {
                    mbar_wait(empty0 + 8 * r.at, r.parity ^ 1, 1);            // (passes at once in the first round)
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx(full0 + 8 * r.at, P * (C::STAGE_W + C::STAGE_A));
                        if (PAIR) {                                           // both CTAs' copies arrive at the first one's barrier
                            const uint32_t bar = tc_map_rank(full0 + 8 * r.at, 0);
                            tma_load_2d_pair(sA + r.at * C::STAGE_A, &map_a, bar, kb * F8_KB, m0);
                            tma_load_2d_pair(sW + r.at * C::STAGE_W, &map_w, bar, kb * F8_KB, n0);
                        } else {
                            tma_load_2d(sA + r.at * C::STAGE_A, &map_a, full0 + 8 * r.at, kb * F8_KB, m0);
                            tma_load_2d(sW + r.at * C::STAGE_W, &map_w, full0 + 8 * r.at, kb * F8_KB, n0);
                        }
                    }
                    __syncwarp();
                }
            }
            f8_drain(empty0, r);
        } else if (warp == 1 && rank == 0) {
            const uint32_t idesc = umma_idesc_e4m3(C::BM, C::BN);
            const uint64_t da0 = make_desc_sw128(sA), dw0 = make_desc_sw128(sW);
            F8Ring<C::STAGES> r;
            F8Ring<C::BUFS> t;
            for (int tile = first; tile < tiles; tile += step) {
                for (int kb = 0; kb < blocks; ++kb, r.next(), t.next()) {
                    const uint64_t da = da0 + r.at * (C::STAGE_A >> 4), dw = dw0 + r.at * (C::STAGE_W >> 4);
                    const uint32_t d = tmem + t.at * C::BN;
                    if (PAIR) {
                        f8_wait_cluster(full0 + 8 * r.at, r.parity, 2);
                        f8_wait_cluster(tempty0 + 8 * t.at, t.parity ^ 1, 2);
                    } else {
                        mbar_wait(full0 + 8 * r.at, r.parity, 2);
                        mbar_wait(tempty0 + 8 * t.at, t.parity ^ 1, 2);
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {                         // 32 codes = 2 descriptor units
                            if (PAIR) umma_f8_pair(d, da + 2 * k, dw + 2 * k, idesc, k > 0 ? 1u : 0u);
                            else umma_f8(d, da + 2 * k, dw + 2 * k, idesc, k > 0 ? 1u : 0u);
                        }
                        if (PAIR) {
                            umma_commit_pair(tfull0 + 8 * t.at);
                            umma_commit_pair(empty0 + 8 * r.at);
                        } else {
                            umma_commit(tfull0 + 8 * t.at);
                            umma_commit(empty0 + 8 * r.at);
                        }
                    }
                    __syncwarp();
                }
            }
        } else if (warp == 2) {
            griddep_wait();
            const int n_blocks = (N + 127) / 128;
            F8Ring<F8_SLOTS> q;
            for (int tile = first; tile < tiles; tile += step) {
                const int m0 = tile % m_tiles * C::BM + rank * 128, nb = tile / m_tiles * P;
                for (int kb = 0; kb < blocks; kb += F8_BATCH, q.next()) {
                    mbar_wait(sempty0 + 8 * q.at, q.parity ^ 1, 1);
                    f8_copy_scales(sScale + q.at * F8_SLOT, sfull0 + 8 * q.at, sc, kb, blocks, m0, M, nb, n_blocks, lane);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");                  // nothing on its way when the CTA leaves
        }
    } else if (GATHER && warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        griddep_wait();
        const int thread = threadIdx.x - 384;
        F8Ring<C::STAGES> r;
        F8Ring<F8_RAWS> in, have;
        int ptile = first, pkb = 0;                                           // two k-blocks ahead
        F8Words words;
        auto request = [&]() {
            if (ptile < tiles) {
                if (pkb == 0) words.start(rows, ptile % m_tiles * C::BM, M, ptile / m_tiles * C::BN, N, K, thread);
                words.copy(sRaw + in.at * F8_RAW, rows, pkb, thread);
                in.next();
                if (++pkb == blocks) { pkb = 0; ptile += step; }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        request();
        request();
        for (int tile = first; tile < tiles; tile += step) {
            const uint64_t offsets = f8_offsets(rows, tile % m_tiles * C::BM, tile / m_tiles * C::BN, thread);
            for (int kb = 0; kb < blocks; ++kb, r.next(), have.next()) {
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                asm volatile("bar.sync 3, 128;" ::: "memory");                // everyone's copies of this k-block are there, and everyone is through with the one before
                request();
                mbar_wait(empty0 + 8 * r.at, r.parity ^ 1, 1);
                f8_place_raw(sRaw + have.at * F8_RAW, sA + r.at * C::STAGE_A, sW + r.at * C::STAGE_W, offsets, thread);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(full0 + 8 * r.at);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        f8_drain(empty0, r);
    } else {
        // (the shares add up to what the CTA was launched with: 40 + 2 x 232 = 3 x 168, with four warps more 40 + 120 + 2 x 176 = 4 x 128)
        if (GATHER) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        griddep_wait();
        constexpr int W = 64 * P;                                             // a thread's columns
        const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
        const uint32_t buf = sStore + (warp - 4) * F8_STORE;
        uint32_t turn = 0;
        const uint32_t columns = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * W);
        const uint32_t factors = sScale + row * (F8_BATCH * 4), factors_w = sScale + (128 + (PAIR ? half : 0)) * (F8_BATCH * 4);
        F8Ring<C::BUFS> t;
        F8Ring<F8_SLOTS> q;
        for (int tile = first; tile < tiles; tile += step) {
            float acc[W];
#pragma unroll
            for (int i = 0; i < W; ++i) acc[i] = 0.f;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int kb = 0; kb < blocks; ++kb, t.next()) {
                if (kb % F8_BATCH == 0) {
                    mbar_wait(sfull0 + 8 * q.at, q.parity, 3);
                    const float4 fa = f8_lds4(factors + q.at * F8_SLOT), fw = f8_lds4(factors_w + q.at * F8_SLOT);
                    f = make_float4(fa.x * fw.x, fa.y * fw.y, fa.z * fw.z, fa.w * fw.w);
                    __syncwarp();
                    f8_arrive0(sempty0 + 8 * q.at, lane);
                    q.next();
                }
                mbar_wait(tfull0 + 8 * t.at, t.parity, 3);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                __syncwarp();                                                 // (the loads of tensor memory are the whole warp's)
                f8_add_block<W>(columns + t.at * C::BN, f.x, acc, [&]() {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    const uint32_t bar = tempty0 + 8 * t.at;
                    if (PAIR) f8_arrive0_cluster(tc_map_rank(bar, 0), lane);
                    else f8_arrive0(bar, lane);
                });
                f = make_float4(f.y, f.z, f.w, 0.f);
            }
            const int m = tile % m_tiles * C::BM + rank * 128, n = tile / m_tiles * C::BN + half * W;
            if constexpr (GATED) {
                // (two places for the largest numbers in turn: whoever writes one again has met everyone behind the reading of it)
                f8_store_gated(acc, gated, sStore + (turn++ & 1) * 1024, half, row, m + row, n, M, N);
            } else {
                f8_store_rows<W, TC>(acc, &map_out, store_by_tma != 0, buf, out, ldc, m + quarter * 32, n, M, N);
            }
        }
        if (lane == 0) tma_store_done();
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) {                                                               // the first CTA's instructions read the other's shared memory, whose barriers they arrive at
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---------------------------------------------------------------- host side
// The shared memory that a kernel needs, set once on every device (twice by two threads at once: it is the same).
template <auto KERNEL, int SMEM>
inline bool f8_configure() {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!done[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return false;
        done[dev].store(true, std::memory_order_relaxed);
    }
    return true;
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
    const int status = launch_status();                                       // (a failed launch leaves nothing behind for the next one to report)
    return e != cudaSuccess ? (int)e : status;
}

inline int f8_sms() {
    int sms = 148, dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    return sms;
}

template <int NT, typename TC>
int launch_float8_few(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, int Z, int w_ready, cudaStream_t stream) {
    CUtensorMap ma, mw;
    if (!f8_make_map(&ma, a, M, K, lda, NT) || !f8_make_map(&mw, w, N, K, ldw, 128)) return AIEN_E_STATE;
    constexpr auto kernel = float8_few_kernel<NT, TC>;
    if (!f8_configure<kernel, F8Few<NT>::SMEM>()) return AIEN_E_STATE;
    const long m_tiles = ((long)M + NT - 1) / NT, n_tiles = ((long)N + 127) / 128;
    if (m_tiles > 65535 || n_tiles > 65535) return AIEN_E_SHAPE;
    return f8_launch(kernel, dim3(Z, (unsigned)m_tiles, (unsigned)n_tiles), 192, F8Few<NT>::SMEM, Z, stream, ma, mw, sc, (TC*)out, ldc, M, N, K, w_ready);
}

template <bool PAIR, bool GATHER, bool GATED, typename TC>
int launch_float8_tiles(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, F8Gated8 gated, cudaStream_t stream) {
    using C = F8Tiles<PAIR, GATHER>;
    constexpr int P = C::P;
    CUtensorMap ma = {}, mw = {}, mo = {};
    if (!GATHER && (!f8_make_map(&ma, a, M, K, lda, 128) || !f8_make_map(&mw, w, N, K, ldw, 128))) return AIEN_E_STATE;
    const bool by_tma = !GATED && ((uintptr_t)out & 15) == 0 && (M == 1 || ldc * sizeof(TC) % 16 == 0);
    if (by_tma && !f8_make_map_out<TC>(&mo, out, M, N, ldc)) return AIEN_E_STATE;
    constexpr auto kernel = float8_tiles_kernel<PAIR, GATHER, GATED, TC>;
    if (!f8_configure<kernel, C::SMEM>()) return AIEN_E_STATE;
    const long m_tiles = ((long)M + C::BM - 1) / C::BM, tiles = m_tiles * (((long)N + C::BN - 1) / C::BN);
    if (tiles > 2147483647L) return AIEN_E_SHAPE;
    const long at_once = f8_sms() / P;
    return f8_launch(kernel, dim3((unsigned)((tiles < at_once ? tiles : at_once) * P)), GATHER ? 512 : 384, C::SMEM, P, stream, ma, mw, mo, (int)by_tma, sc,
                     (TC*)out, ldc, M, N, K, (int)m_tiles, (int)tiles, F8Rows{(const uint8_t*)a, lda, (const uint8_t*)w, ldw}, gated);
}

// The product's form, by the time that each would take (us; measured with K of 4,096 and 12,288 on rows of 8 to 4,096, with one to three waves):
//   in tiles of 128 x 128      3.2 and 0.28 a k-block and wave of one tile an SM
//   in pairs, 256 x 256        3.0 and 0.44 a k-block and wave of one tile a pair of SMs
//   few rows, 128 x NT         2.3, shared by a cluster of 2, 4 or 8 4.6, 3.7 or 4.1 (with 64 columns 2.2 more), and a k-block 0.23 where the CTAs are
//                              few (with 64 columns, whose ring is shorter, 0.39), else W's bytes at 6.5 TB/s; more than 64 rows in tiles of 64
//                              0.002 a CTA, which L2 and the reading of tensor memory take; two CTAs an SM
// 256 x 4,096 x 4,096: 11.8 us in tiles, 15.5 in pairs, 16.6 in the form for few rows; 128 x 4,096 x 12,288: 28.2, 37.0 and 17.8;
// 1,024 x 4,096 x 4,096: 20.7, 17.1 and 36.8; 67 x 1,000 x 2,064: 8.8 in tiles and 7.3 in the form for few rows.  8 rows by clusters of 1, 2, 4 and 8:
// 4,096 x 4,096 9.7, 8.2, 6.2 and 6.6; 6,144 x 4,096 10.2, 9.1, 7.7 and 10.4; 4,096 x 12,288 24.4, 15.5, 11.4 and 11.6; 24,576 x 4,096 19.6, 24.4, 23.2
// and 31.7.
struct F8Plan {
    int form, Z;              // columns of the form for few rows (16, 32 or 64), 1 tiles, 2 pairs; CTAs that share K
};
inline F8Plan f8_plan(int M, int N, int K) {
    const long sms = f8_sms(), blocks = ((long)K + F8_KB - 1) / F8_KB, n_tiles = ((long)N + 127) / 128;
    const int nt = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    const long few = ((long)M + nt - 1) / nt * n_tiles;
    F8Plan best = {nt, 1};
    double least = 1e30;
    for (int Z = 1; Z <= 8 && Z <= blocks; Z *= 2) {
        const long ctas = few * Z, at_once = ctas < 2 * sms ? ctas : 2 * sms;
        const double busy = at_once * (M <= 64 ? 0.0025 : 0.002), least_each = nt == 64 ? 0.39 : 0.23, each = busy > least_each ? busy : least_each;
        const double t = (Z == 1 ? 2.3 : Z == 2 ? 4.6 : Z == 4 ? 3.7 : 4.1) + (nt == 64 ? 2.2 : 0.) + (double)((blocks + Z - 1) / Z) * each * (double)((ctas + 2 * sms - 1) / (2 * sms));
        if (t < least) { least = t; best.Z = Z; }
    }
    if (n_tiles > 65535) return F8Plan{1, 1};                                 // beyond the grid of the form for few rows
    if (M <= 64) return best;
    const long alone = ((long)M + 127) / 128 * n_tiles, pairs = ((long)M + 255) / 256 * (((long)N + 255) / 256);
    const double t1 = 3.2 + 0.28 * blocks * (double)((alone + sms - 1) / sms), t2 = 3.0 + 0.44 * blocks * (double)((pairs + sms / 2 - 1) / (sms / 2));
    if (least <= t1 && least <= t2) return best;
    return t1 <= t2 ? F8Plan{1, 1} : F8Plan{2, 1};
}

// every row of codes starts on a 16-byte border
inline bool f8_whole_rows(const void* a, long lda, const void* w, long ldw, int M, int N) {
    return (((uintptr_t)a | (uintptr_t)w) & 15) == 0 && (M == 1 || lda % 16 == 0) && (N == 1 || ldw % 16 == 0);
}

template <typename TC>
int launch_float8(const void* a, long lda, const void* w, long ldw, F8Scales sc, void* out, long ldc, int M, int N, int K, int w_ready, cudaStream_t stream) {
    if (!f8_whole_rows(a, lda, w, ldw, M, N)) return launch_float8_tiles<false, true, false, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, F8Gated8{}, stream);
    const F8Plan plan = f8_plan(M, N, K);
#define F8_FEW(NT) return launch_float8_few<NT, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, plan.Z, w_ready, stream)
    if (plan.form == 16) F8_FEW(16);
    if (plan.form == 32) F8_FEW(32);
    if (plan.form == 64) F8_FEW(64);
#undef F8_FEW
    if (plan.form == 1) return launch_float8_tiles<false, false, false, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, F8Gated8{}, stream);
    return launch_float8_tiles<true, false, false, TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, F8Gated8{}, stream);
}

}  // namespace aien

// a [M, K] and w [N, K] codes, rows lda and ldw bytes apart; sa [ceil(K / 128), M] (lds numbers apart); sw [ceil(N / 128), ceil(K / 128)] (ldsw
// numbers apart); out [M, N], rows ldc numbers apart.  w_ready: w and its scales were written by nothing that an unfinished kernel ahead in the stream
// does, so that they may be requested before it is done.
AIEN_API int aien_matmul_float8(const void* a, long lda, const float* sa, long lds, const void* w, long ldw, const float* sw, long ldsw,
                                   void* out, int c_dt, long ldc, int M, int N, int K, int w_ready, cudaStream_t stream) {
    using namespace aien;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return AIEN_E_SHAPE;
    const F8Scales sc{sa, lds, sw, ldsw};
    AIEN_DISPATCH_DTYPE(c_dt, TC, return (launch_float8<TC>(a, lda, w, ldw, sc, out, ldc, M, N, K, w_ready, stream)));
}

// The product with act(gate) * up of its columns in 8 bits as its result: W's rows are gate and up in runs of 8 (N counts both), codes [M, N / 2], rows ldq
// bytes apart, scales [ceil(N / 256), M], lds8 numbers apart.  In pairs of CTAs; rows of codes on 16-byte borders.
AIEN_API int aien_matmul_swiglu_float8(const void* a, long lda, const float* sa, long lds, const void* w, long ldw, const float* sw, long ldsw,
                                       void* codes, long ldq, float* scales, long lds8, int gelu, int M, int N, int K, cudaStream_t stream) {
    using namespace aien;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (N & 15)) return AIEN_E_SHAPE;
    if (!f8_whole_rows(a, lda, w, ldw, M, N)) return AIEN_E_ALIGN;
    return launch_float8_tiles<true, false, true, __nv_bfloat16>(a, lda, w, ldw, F8Scales{sa, lds, sw, ldsw}, nullptr, 0, M, N, K,
                                                                 F8Gated8{(uint8_t*)codes, ldq, scales, lds8, gelu}, stream);
}

// Whether that is the product's own form at this size, so that one kernel takes less than two.
AIEN_API int aien_matmul_swiglu_float8_supports(int M, int N, int K) {
    return M > 0 && N > 0 && K > 0 && N % 16 == 0 && aien::f8_plan(M, N, K).form == 2;
}
