// dense_e4m3.cu - matrix product over e4m3 operands with a float32 scale per
// block of 128 (rows of x: 1 x 128; weights: 128 x 128) on the 5th-generation
// tensor cores.
//
//     y[m][n] = sum_b xs[b][m] ws[n / 128][b] (sum_{k in b} xq[m][k] wq[n][k])  (+ bias[n])
//
// The inner sum, 128 products, is one accumulation of four tcgen05.mma
// (kind::f8f6f4, 32 of K each) into a fresh TMEM accumulator; the outer one
// runs in float32 registers: the epilogue warps read each block's partial
// from TMEM and add it times the block's scale, while the MMAs of the next
// blocks fill the other accumulators.  Rows and columns past M, N and K are
// zero-filled by TMA and never stored.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "act16.cuh"
#include "clusters.cuh"
#include "e4m3.cuh"
#include "gemm.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace rg {
namespace {

template <Elem O>
__device__ __forceinline__ void store_y(void* y, int64_t at, float v) {
    if constexpr (O == Elem::kF32)
        static_cast<float*>(y)[at] = v;
    else
        static_cast<uint16_t*>(y)[at] = from_f32<O == Elem::kF16>(v);
}

// ---------------------------------------------------------------------------
// Few rows of x: weight rows on the M side of the MMA.  A CTA owns 128 weight
// rows (one weight block, so its weight scale is one number per block of K)
// and NT rows of x, over its share of K; the shares of a cluster's CTAs are
// joined through distributed shared memory, in rank order.  Such products
// wait for the weights: two CTAs an SM keep two times four stages of 16 KB of
// them in flight (37 x 8192 x 4096: 10.2 us, 34 MB of weights from L2; the first
// bytes arrive after 1.5 us, the joins take 2.5).  The tensor memory of as many
// CTAs as shared memory lets on an SM never exceeds it, so none waits for
// another's.  Roles (256 threads):
//   warp 0     TMA producer: 128 weight rows and NT x rows of each k-block;
//   warp 1     MMA issuer, four MMAs per k-block into one of ACC accumulators;
//   warp 2     TMEM allocator, then the scales of each k-block into a ring in
//              shared memory (asynchronous copies: loads into registers, one
//              k-block at a time, held everything else up);
//   warps 4-7  accumulation, thread = weight row = TMEM lane, NT sums each.
template <int NT>
struct ThinShape {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = NT * 128;
    static constexpr int STAGES = 4;
    static constexpr int ACC = 4;
    static constexpr uint32_t TMEM_COLS = ACC * NT;
    static constexpr int SR = 8;           // ring of scales
    static constexpr int SLOT = NT + 4;    // x scales, then the weight scale
    static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES) + SR * SLOT * 4 + 1024 + 512;
    static constexpr int THREADS = 256;
    static_assert(STAGES * (A_BYTES + B_BYTES) >= NT * 512, "the sums of a CTA take the place of its stages");
    static_assert(228 * 1024 / SMEM * TMEM_COLS <= 512, "no CTA waits for another's tensor memory");
};

template <int NT, Elem O>
__global__ void __launch_bounds__(256, 2)
    dense_e4m3_thin_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           DenseE4Params p, int split) {
    using S = ThinShape<NT>;
    constexpr int STAGES = S::STAGES, ACC = S::ACC, SR = S::SR;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * S::A_BYTES;
    float* sScale = reinterpret_cast<float*>(sB + STAGES * S::B_BYTES);  // [SR][SLOT]
    uint64_t* full = reinterpret_cast<uint64_t*>(sScale + SR * S::SLOT);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + ACC;
    uint64_t* cfull = tempty + ACC;
    uint64_t* cempty = cfull + SR;
    uint64_t* drain = cempty + SR;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int kblocks = (p.K + kE4Block - 1) / kE4Block;
    const int rank = blockIdx.x % split;  // its share of K: blocks [k0, k0 + nk)
    const int k0 = static_cast<int>(static_cast<int64_t>(kblocks) * rank / split);
    const int nk = static_cast<int>(static_cast<int64_t>(kblocks) * (rank + 1) / split) - k0;
    const int nb = blockIdx.x / split, n0 = nb * 128, m0 = blockIdx.y * NT;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < ACC; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 4);
        }
        for (int s = 0; s < SR; ++s) {
            mbar_init(&cfull[s], 32);  // the copies of every lane of the scale warp
            mbar_init(&cempty[s], 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, S::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    pdl_wait();
    const uint32_t tmem = *tmem_slot;

    float sum[NT];
    if (warp == 0) {
        int issued = 0;
        for (int kb = 0; kb < nk; ++kb) {
            const int s = kb % STAGES;
            if (!mbar_wait_warp(&empty[s], ((kb / STAGES) & 1) ^ 1, p.status, abort_flag)) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(&full[s], S::A_BYTES + S::B_BYTES);
                tma_load_2d(sA + s * S::A_BYTES, &tmW, &full[s], (k0 + kb) * 128, n0);
                tma_load_2d(sB + s * S::B_BYTES, &tmX, &full[s], (k0 + kb) * 128, m0);
            }
            __syncwarp();
            issued = kb + 1;
        }
        // every load issued has landed before the CTA may exit
        for (int kb = issued > STAGES ? issued - STAGES : 0; kb < issued; ++kb)
            mbar_drain(&full[kb % STAGES], (kb / STAGES) & 1);
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_e4m3(128, NT);
        const uint64_t ad0 = sdesc_k128(smem_u32(sA)), bd0 = sdesc_k128(smem_u32(sB));
        bool issued = false;
        for (int kb = 0; kb < nk; ++kb) {
            const int s = kb % STAGES, a = kb % ACC;
            if (!mbar_wait_warp(&tempty[a], ((kb / ACC) & 1) ^ 1, p.status, abort_flag) ||
                !mbar_wait_warp(&full[s], (kb / STAGES) & 1, p.status, abort_flag))
                break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t ad = ad0 + s * (S::A_BYTES / 16), bd = bd0 + s * (S::B_BYTES / 16);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + a * NT, ad + 2 * k, bd + 2 * k, idesc, k > 0);
                umma_commit(&empty[s]);
                umma_commit(&tfull[a]);
            }
            __syncwarp();
            issued = true;
        }
        if (issued) {
            if (elect_one()) umma_commit(drain);
            mbar_drain(drain, 0);
        }
    } else if (warp == 2) {
        const float* xs = p.x_scale + k0 * p.ld_xs + m0 + lane;
        const float* ws = p.w_scale + static_cast<int64_t>(nb) * kblocks + k0;
        for (int kb = 0; kb < nk; ++kb) {
            const int c = kb % SR;
            if (!mbar_wait_warp(&cempty[c], ((kb / SR) & 1) ^ 1, p.status, abort_flag)) break;
            float* to = sScale + c * S::SLOT;
#pragma unroll
            for (int i = 0; i < NT; i += 32)
                if (lane + i < NT) {  // rows past the end: zeros
                    const bool in = m0 + lane + i < p.M;
                    cp_async_f32(to + lane + i, in ? xs + i : p.x_scale, in);
                }
            if (lane == 0) cp_async_f32(to + NT, ws + kb, true);
            cp_async_arrive(&cfull[c]);
            xs += p.ld_xs;
        }
        cp_async_wait_all();
    } else if (warp >= 4) {
        const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
#pragma unroll
        for (int i = 0; i < NT; ++i) sum[i] = 0.f;
        bool ok = true;
        for (int kb = 0; kb < nk; ++kb) {
            const int a = kb % ACC, c = kb % SR;
            if (!mbar_wait_warp(&cfull[c], (kb / SR) & 1, p.status, abort_flag) ||
                !mbar_wait_warp(&tfull[a], (kb / ACC) & 1, p.status, abort_flag)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const float4* sc = reinterpret_cast<const float4*>(sScale + c * S::SLOT);
            const float w = sScale[c * S::SLOT + NT];
#pragma unroll
            for (int h = 0; h < NT / 16; ++h) {
                uint32_t t[16];
                tmem_ld16(tmem + lane_addr + a * NT + h * 16, t);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 s4 = sc[h * 4 + i];
                    float* to = sum + h * 16 + 4 * i;
                    to[0] = fmaf(__uint_as_float(t[4 * i + 0]), s4.x * w, to[0]);
                    to[1] = fmaf(__uint_as_float(t[4 * i + 1]), s4.y * w, to[1]);
                    to[2] = fmaf(__uint_as_float(t[4 * i + 2]), s4.z * w, to[2]);
                    to[3] = fmaf(__uint_as_float(t[4 * i + 3]), s4.w * w, to[3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&tempty[a]);
                mbar_arrive(&cempty[c]);
            }
        }
        if (!ok) sum[0] = 0.f;  // the status says that the result is not one
    }
    // Every role of every CTA is done and the stages' memory is free: it takes
    // the sums, four rows of x to a float4, [split][NT / split / 4][128]: each
    // CTA's share of the tile's rows from all of them (stores to the owner's
    // memory, which nothing waits for).
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, S::TMEM_COLS);
    }
    const int lg = __ffs(NT / 4 / split) - 1, per = 1 << lg;  // groups of four rows of a CTA
    float4* part = reinterpret_cast<float4*>(sA);
    const int col = threadIdx.x & 127, n = n0 + col;
    if (split > 1) {
        cluster_sync();
        if (warp >= 4) {
            const uint32_t to = smem_u32(part + rank * per * 128 + col);
#pragma unroll
            for (int i = 0; i < NT / 4; ++i)
                if (m0 + 4 * i < p.M)
                    st_shared_cluster(mapa_shared(to + (i & (per - 1)) * 2048, i >> lg), sum[4 * i], sum[4 * i + 1],
                                      sum[4 * i + 2], sum[4 * i + 3]);
        }
        cluster_sync();
    } else {
        if (warp >= 4) {
#pragma unroll
            for (int i = 0; i < NT / 4; ++i)
                part[i * 128 + col] = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
        }
        __syncthreads();
    }
    const float b = p.bias && n < p.N ? __ldg(p.bias + n) : 0.f;
    float amax = 0.f;
    for (int i = threadIdx.x >> 7; i < per && n < p.N; i += 2) {
        const int m = m0 + 4 * (rank * per + i);
        if (m >= p.M) break;
        float4 f[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < split) f[r] = part[(r * per + i) * 128 + col];
        float4 v = f[0];
#pragma unroll
        for (int r = 1; r < 8; ++r)
            if (r < split) {
                v.x += f[r].x;
                v.y += f[r].y;
                v.z += f[r].z;
                v.w += f[r].w;
            }
        const float out[4] = {v.x + b, v.y + b, v.z + b, v.w + b};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m + j < p.M) {
                store_y<O>(p.y, (m + j) * p.ldy + n, out[j]);
                amax = fmaxf(amax, fabsf(out[j]));
            }
    }
    if (O == Elem::kF16 && amax > 65504.0f) atomicOr(p.status, kStatusF16Overflow);
}

// ---------------------------------------------------------------------------
// Large products: persistent CTA pairs (clusters of 2, cta_group::2) on tiles
// of 256 x BN.  Per k-block the pair's four MMAs fill one of the TMEM
// accumulators, which the accumulation warps read back.  At BN = 256 that is 512
// cycles of the tensor core against 128 x 256 values to read, scale and add per
// CTA, which bounds the kernel: 16384 x 4096 x 4096 takes 243 us (2265 TFLOP/s;
// 320 us in a sustained loop, where the card lowers its clock to some 1.45
// GHz), 162 us with the handshake and the accumulation taken out, 178 without
// the reading and the additions alone.  What carried it there: MMAs issued from
// warp-uniform code (elect_one; half the time of a lane's branch), arrivals
// without release at cluster scope, scales by asynchronous copies, and registers
// enough for the sums.  Roles (384 threads):
//   warp 0      TMA producer of its CTA's 128 rows of x and BN / 2 of w;
//   warp 1      (even CTA) MMA issuer;
//   warp 2      TMEM allocator;
//   warp 3      scales: each k-block's 128 row scales and two weight scales
//               into a ring in shared memory, by asynchronous copies;
//   warps 4-11  accumulation: warp (4 + 4 h + q) owns rows [32 q, +32) and
//               columns [h BN / 2, +BN / 2), thread = row, BN / 2 fp32 sums in
//               registers (the control warps give registers up for them).  A
//               half of the columns lies within one weight block, so one
//               factor per thread serves a k-block.
template <int BN>
struct WideShape {
    static constexpr int HALF = BN / 2;
    static constexpr int A_BYTES = 128 * 128, B_BYTES = HALF * 128;
    static constexpr int STAGES = BN == 256 ? 5 : 7;
    static constexpr int ACC = 512 / BN;
    static constexpr int WARPS = 8;
    static constexpr int BOXES = 4096;  // a warp's 32 x 32 boxes: one of fp32 or two of 16 bits
    static constexpr int SR = 8;        // ring of scales, 2 x 128 each
    static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES) + WARPS * BOXES + SR * 1024 + 1024 + 512;
    static constexpr int THREADS = 128 + 32 * WARPS;
    // 128 * 24 + 256 * 240 = 384 * 168; with 232 for the sums their pairs are
    // moved about (16384 x 4096 x 4096: 255 against 243 us); 20 to 36 bytes are spilled
    static constexpr int CONTROL_REGS = 24, SUM_REGS = 240;
    static_assert(SMEM <= 232448, "shared memory");
};

// RAGGED: the rows of y, written by TMA, end between 16 bytes.  TMA writes whole
// ones, zeros behind the row, so that their last box goes out by plain stores (a
// kernel of its own: as a test in the other it moved registers about in the loop
// over K, 16384 x 4096 x 4096 276 against 267 us; y without TMA took 348 us where
// N = 4100).
template <int BN, Elem O, bool RAGGED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(384, 1)
    dense_e4m3_wide_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const __grid_constant__ CUtensorMap tmY, DenseE4Params p, bool tma_out) {
    using S = WideShape<BN>;
    constexpr int STAGES = S::STAGES, ACC = S::ACC, HALF = S::HALF, SR = S::SR;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * S::A_BYTES;
    uint8_t* boxes = sB + STAGES * S::B_BYTES;
    float* sScale = reinterpret_cast<float*>(boxes + S::WARPS * S::BOXES);  // [SR][128 rows, 2 weight blocks]
    uint64_t* full = reinterpret_cast<uint64_t*>(sScale + SR * 130);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + ACC;
    uint64_t* cfull = tempty + ACC;
    uint64_t* cempty = cfull + SR;
    uint64_t* drain = cempty + SR;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();  // 0: the CTA that issues the MMAs
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int n_tiles = (p.N + BN - 1) / BN;
    const int num_tiles = (p.M + 255) / 256 * n_tiles;
    const int kblocks = (p.K + kE4Block - 1) / kE4Block;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < ACC; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 2 * S::WARPS);  // the accumulation warps of both CTAs
        }
        for (int s = 0; s < SR; ++s) {
            mbar_init(&cfull[s], 32);
            mbar_init(&cempty[s], S::WARPS);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
        if (tma_out) tma_prefetch_desc(&tmY);
    }
    if (warp == 2) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    pdl_trigger();
    pdl_wait();
    const uint32_t tmem = *tmem_slot;
    const uint32_t full_lead = mapa_shared(smem_u32(full), 0);
    const uint32_t tempty_lead = mapa_shared(smem_u32(tempty), 0);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::CONTROL_REGS));
        if (warp == 0) {
            int stage = 0;
            uint32_t phase = 0;
            int issued = 0;  // up to the ring's depth
            bool ok = true;
            for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
                const int row = tile / n_tiles * 256 + static_cast<int>(rank) * 128;
                const int col = tile % n_tiles * BN + static_cast<int>(rank) * HALF;
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait_warp(&empty[stage], phase ^ 1, p.status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        // both CTAs' loads complete on the even CTA's barrier
                        if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * (S::A_BYTES + S::B_BYTES));
                        tma_load_2d_pair(sA + stage * S::A_BYTES, &tmX, full_lead + 8 * stage, kb * 128, row);
                        tma_load_2d_pair(sB + stage * S::B_BYTES, &tmW, full_lead + 8 * stage, kb * 128, col);
                    }
                    __syncwarp();
                    issued = min(issued + 1, STAGES);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // the even CTA sees every load of both CTAs land
            for (; issued > 0; --issued) {
                if (--stage < 0) {
                    stage = STAGES - 1;
                    phase ^= 1;
                }
                if (rank == 0) mbar_drain(&full[stage], phase);
            }
        } else if (warp == 1 && rank == 0) {
            constexpr uint32_t idesc = idesc_e4m3(256, BN);
            const uint32_t ad0 = static_cast<uint32_t>(sdesc_k128(smem_u32(sA)));
            const uint32_t bd0 = static_cast<uint32_t>(sdesc_k128(smem_u32(sB)));
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool issued = false, ok = true;
            for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1, p.status, abort_flag) ||
                        !mbar_wait_warp(&full[stage], phase, p.status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t ad = ad0 + stage * (S::A_BYTES / 16), bd = bd0 + stage * (S::B_BYTES / 16);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f8_pair(tmem + acc * BN, ad + 2 * k, bd + 2 * k, idesc, k > 0);
                        umma_commit_pair_mc(smem_u32(&empty[stage]), 0x3);
                        umma_commit_pair_mc(smem_u32(&tfull[acc]), 0x3);
                    }
                    __syncwarp();
                    issued = true;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                    if (++acc == ACC) {
                        acc = 0;
                        acc_phase ^= 1;
                    }
                }
            }
            if (issued) {
                if (elect_one()) umma_commit_pair(smem_u32(drain));
                mbar_drain(drain, 0);
            }
        } else if (warp == 3) {
            const int nblocks = (p.N + kE4Block - 1) / kE4Block;
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
                const int row = tile / n_tiles * 256 + static_cast<int>(rank) * 128 + lane;
                const int nb = (tile % n_tiles * BN + (lane & 1) * HALF) / kE4Block;
                const bool in_n = nb < nblocks;
                const float* xs = p.x_scale + row;
                const float* ws = p.w_scale + (in_n ? static_cast<int64_t>(nb) * kblocks : 0);
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait_warp(&cempty[slot], phase ^ 1, p.status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    float* to = sScale + slot * 130;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // rows past the end: zeros
                        const bool in = row + 32 * i < p.M;
                        cp_async_f32(to + lane + 32 * i, in ? xs + 32 * i : p.x_scale, in);
                    }
                    if (lane < 2) cp_async_f32(to + 128 + lane, ws + kb, in_n);
                    cp_async_arrive(&cfull[slot]);
                    xs += p.ld_xs;
                    if (++slot == SR) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
            // every copy has landed before the CTA may exit
            cp_async_wait_all();
        }
        // The control warps gave registers up: nothing is shared with the
        // accumulation warps' code from here on but the barrier.
        __syncwarp();
        tc_fence_before();
        cluster_sync();
        if (warp == 2) {
            tc_fence_after();
            tmem_dealloc_pair(tmem, 512);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::SUM_REGS));
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;
        uint8_t* box = boxes + ew * S::BOXES;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        int acc = 0, slot = 0, stores = 0;
        uint32_t acc_phase = 0, slot_phase = 0;
        bool ok = true;
        for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
            const int row0 = tile / n_tiles * 256 + static_cast<int>(rank) * 128 + quarter * 32;
            const int col0 = tile % n_tiles * BN + half * HALF;
            const int row = row0 + lane;
            uint64_t sum[HALF / 2];
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) sum[i] = 0;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!mbar_wait_warp(&cfull[slot], slot_phase, p.status, abort_flag)) {
                    ok = false;
                    break;
                }
                const float s = sScale[slot * 130 + quarter * 32 + lane] * sScale[slot * 130 + 128 + half];
                const uint64_t s2 = pair_of(s, s);
                if (!mbar_wait_warp(&tfull[acc], acc_phase, p.status, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t ta = tmem + lane_addr + acc * BN + half * HALF;
                // 64 columns at a time: the latency of a load from tensor memory, long
                // while products write there, is met twice instead of eight times
                constexpr int C = HALF < 64 ? HALF : 64;
                uint32_t t[C];
#pragma unroll
                for (int c = 0; c < HALF; c += C) {
#pragma unroll
                    for (int i = 0; i < C; i += 32) tmem_ld32(ta + c + i, *reinterpret_cast<uint32_t(*)[32]>(&t[i]));
                    tmem_ld_wait();
                    if (c + C == HALF) {  // all of it is in registers: the next MMAs may have the accumulator
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive_cluster_relaxed(tempty_lead + 8 * acc);
                            mbar_arrive(&cempty[slot]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < C / 2; ++i)
                        sum[c / 2 + i] = fma_pair(pair_of(__uint_as_float(t[2 * i]), __uint_as_float(t[2 * i + 1])), s2,
                                                  sum[c / 2 + i]);
                }
                if (++acc == ACC) {
                    acc = 0;
                    acc_phase ^= 1;
                }
                if (++slot == SR) {
                    slot = 0;
                    slot_phase ^= 1;
                }
            }
            if (!ok) break;
#pragma unroll
            for (int c = 0; c < HALF / 32; ++c) {
                const int c0 = col0 + c * 32;
                if (c0 >= p.N || row0 >= p.M) break;  // warp-uniform
                float v[32];
#pragma unroll
                for (int i = 0; i < 16; ++i) split_pair(sum[c * 16 + i], v[2 * i], v[2 * i + 1]);
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c0 + i < p.N) v[i] += __ldg(p.bias + c0 + i);
                }
                if (O == Elem::kF16) {
                    float amax = 0.f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));
                    if (row < p.M && amax > 65504.0f) atomicOr(p.status, kStatusF16Overflow);
                }
                if (tma_out && (!RAGGED || c0 + 32 <= p.N)) {
                    // the store that last read this box has left it
                    uint8_t* b = O == Elem::kF32 ? box : box + (stores & 1) * 2048;
                    if (lane == 0) {
                        if (O == Elem::kF32) bulk_wait_read<0>();
                        else bulk_wait_read<1>();
                    }
                    __syncwarp();
                    if constexpr (O == Elem::kF32) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(b + ((lane * 128 + i * 16) ^ ((lane & 7) << 4))) =
                                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<uint4*>(b + ((lane * 64 + i * 16) ^ (((lane >> 1) & 3) << 4))) =
                                make_uint4(pack2<O == Elem::kF16>(v[8 * i], v[8 * i + 1]),
                                           pack2<O == Elem::kF16>(v[8 * i + 2], v[8 * i + 3]),
                                           pack2<O == Elem::kF16>(v[8 * i + 4], v[8 * i + 5]),
                                           pack2<O == Elem::kF16>(v[8 * i + 6], v[8 * i + 7]));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmY, b, c0, row0);
                        bulk_commit();
                    }
                    ++stores;
                } else {
                    // rows of y that TMA cannot address: through shared memory, so
                    // that a warp writes 32 neighbours of one row
                    if (RAGGED) {
                        if (lane == 0) bulk_wait_read<0>();
                        __syncwarp();
                    }
                    float* f = reinterpret_cast<float*>(box);
#pragma unroll
                    for (int i = 0; i < 32; ++i) f[lane * 32 + (i ^ lane)] = v[i];
                    __syncwarp();
                    for (int r = 0; r < 32; ++r)
                        if (row0 + r < p.M && c0 + lane < p.N)
                            store_y<O>(p.y, (row0 + r) * p.ldy + c0 + lane, f[r * 32 + (lane ^ r)]);
                    __syncwarp();
                }
            }
        }
        if (tma_out && lane == 0) bulk_wait_read<0>();
        __syncwarp();
        tc_fence_before();
        cluster_sync();
    }
}

template <typename K>
cudaError_t allow_smem(K kern, int bytes, unsigned& configured) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 32 && (__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & (1u << dev))) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 32) __atomic_fetch_or(&configured, 1u << dev, __ATOMIC_RELEASE);
    return e;
}

// K is split over up to eight CTAs (of at least four rows each in the join)
// while they all run at once.  That is two an SM, which the occupancy query does
// not know (it counts one CTA an SM for kernels that allocate tensor memory), so
// that the bound is a measured one: clusters of four and eight leave a tenth of
// the places empty, as they do not cross GPCs (of 256 CTAs all ran at once, of
// 288 and 296 some waited: 100 x 4736 x 16384 47 us over four, 39 over two).
int thin_split(const DenseE4Params& p, int nt, int num_sms) {
    const int64_t tiles = static_cast<int64_t>((p.N + 127) / 128) * ((p.M + nt - 1) / nt);
    const int kblocks = (p.K + kE4Block - 1) / kE4Block;
    int split = 1;
    for (int s = 2; s <= 8 && s <= nt / 4 && s <= kblocks; s *= 2)
        if (s * tiles <= (s == 2 ? 2 * num_sms : 2 * num_sms * 9 / 10)) split = s;
    return split;
}

template <int NT, Elem O>
cudaError_t launch_thin(const DenseE4Params& p, int split, cudaStream_t st) {
    using S = ThinShape<NT>;
    static unsigned configured = 0;
    auto kern = dense_e4m3_thin_kernel<NT, O>;
    cudaError_t e = allow_smem(kern, S::SMEM, configured);
    if (e != cudaSuccess) return e;
    CUtensorMap tw, tx;
    if (!make_kmajor_tmap(&tw, p.wq, 1, p.N, p.K, p.ldw, 128) || !make_kmajor_tmap(&tx, p.xq, 1, p.M, p.K, p.ldx, NT))
        return cudaErrorInvalidValue;
    const int tiles_n = (p.N + 127) / 128, tiles_m = (p.M + NT - 1) / NT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles_n * split, tiles_m);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, tw, tx, p, split);
}

template <int BN, Elem O, bool RAGGED>
cudaError_t launch_wide_as(const DenseE4Params& p, const CUtensorMap* out, cudaStream_t st) {
    using S = WideShape<BN>;
    static ClusterCounts known = {};
    auto kern = dense_e4m3_wide_kernel<BN, O, RAGGED>;
    int pairs = 0;  // one per tile slot: as many as can be resident at once
    cudaError_t e = clusters_at_once(kern, S::THREADS, S::SMEM, 2, known, pairs);
    if (e != cudaSuccess) return e;
    CUtensorMap tx, tw;
    if (!make_kmajor_tmap(&tx, p.xq, 1, p.M, p.K, p.ldx, 128) ||
        !make_kmajor_tmap(&tw, p.wq, 1, p.N, p.K, p.ldw, S::HALF))
        return cudaErrorInvalidValue;
    const bool tma_out = out != nullptr;
    const CUtensorMap ty = out ? *out : tx;  // not read without
    const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + BN - 1) / BN);
    const dim3 grid(2 * static_cast<unsigned>(tiles < pairs ? tiles : pairs));
    return launch_pdl(kern, grid, dim3(S::THREADS), S::SMEM, st, tx, tw, ty, p, tma_out);
}

template <int BN, Elem O>
cudaError_t launch_wide(const DenseE4Params& p, cudaStream_t st) {
    CUtensorMap ty;
    if (!make_epilogue_tmap(&ty, p.y, O == Elem::kF32, O == Elem::kF16, p.M, p.N, p.ldy))
        return launch_wide_as<BN, O, false>(p, nullptr, st);
    if (p.N % (O == Elem::kF32 ? 4 : 8) == 0) return launch_wide_as<BN, O, false>(p, &ty, st);
    return launch_wide_as<BN, O, true>(p, &ty, st);
}

// Up to 32 rows the weights' bytes count, and the thin kernel spreads them over
// the SMs.  Above, the kernel and tile width whose waves are estimated to take
// less, in microseconds a k-block: a pair's tile of 256 columns 0.50, of 128
// 0.33; thin tiles of 64 rows 0.5 while each has an SM to itself, two an SM
// 0.75, and 3 for their start and join (thin against wide: 100 x 4096 x 4096
// 16 and 18.5 us, 100 x 16384 x 16384 90 and 76, 200 x 1024 x 16384 22 and 45,
// 200 x 4096 x 4096 22.5 and 18.5, 300 x 1024 x 4096 16 and 18.5; widths 128 and
// 256: 512 x 4096 x 4096 21 and 27, 1024 x 4096 x 4096 31 and 29).
template <Elem O>
cudaError_t launch_out(const DenseE4Params& p, int num_sms, cudaStream_t st) {
    if (p.M <= 16) return launch_thin<16, O>(p, thin_split(p, 16, num_sms), st);
    if (p.M <= 32) return launch_thin<32, O>(p, thin_split(p, 32, num_sms), st);
    const int64_t kblocks = (p.K + kE4Block - 1) / kE4Block;
    const int64_t pairs = num_sms / 2, rows = (p.M + 255) / 256;
    const int64_t waves256 = (rows * ((p.N + 255) / 256) + pairs - 1) / pairs;
    const int64_t waves128 = (rows * ((p.N + 127) / 128) + pairs - 1) / pairs;
    const float wide256 = 0.50f * static_cast<float>(waves256), wide128 = 0.33f * static_cast<float>(waves128);
    const int64_t tiles_m = (p.M + 63) / 64;
    if (tiles_m <= 65535) {
        const int split = thin_split(p, 64, num_sms);
        const int64_t ctas = tiles_m * ((p.N + 127) / 128) * split;
        const int64_t waves = (ctas + 2 * num_sms - 1) / (2 * num_sms);
        const float block = ctas <= num_sms ? 0.5f : 0.75f * static_cast<float>(waves);
        const float thin = 3.0f + block * static_cast<float>((kblocks + split - 1) / split);
        if (thin <= std::min(wide256, wide128) * static_cast<float>(kblocks)) return launch_thin<64, O>(p, split, st);
    }
    if (wide128 < wide256) return launch_wide<128, O>(p, st);
    return launch_wide<256, O>(p, st);
}

}  // namespace

cudaError_t launch_dense_e4m3(Elem out, const DenseE4Params& p, int num_sms, cudaStream_t st) {
    switch (out) {
    case Elem::kF32: return launch_out<Elem::kF32>(p, num_sms, st);
    case Elem::kF16: return launch_out<Elem::kF16>(p, num_sms, st);
    case Elem::kBF16: return launch_out<Elem::kBF16>(p, num_sms, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace rg
