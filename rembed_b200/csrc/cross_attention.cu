// cross_attention.cu - cross attention on the 5th-generation tensor cores:
// tiles of 128 query rows of one (sequence, query head) against blocks of BKV
// keys, one pass with the running maximum and sum of the softmax.
//
// Roles (head dims up to 128: two tiles a CTA, 384 threads; 256: one, 256):
//   warp 0     TMA producer: the query tiles once, then K and V blocks through
//              two stages each.  In the last block, which may reach past the
//              sequence's end, the rows of V behind it that share a
//              16-key MMA step with it are overwritten with zeros (they may
//              hold anything: 0 * NaN would reach the output);
//   warp 1     MMA issuer: S = Q K^T into tensor memory, O += P V with P read
//              from tensor memory, where it takes the place of its S;
//   warp 2     TMEM allocator;
//   warps 4..  softmax, four warps a tile, thread = query row = TMEM lane.
// With two tiles the softmax of one runs under the MMAs of the other; the one
// tile of head dim 256 has two S buffers instead.  The tensor core finishes a
// thread's MMAs in order, so a block's S being ready implies that the tile's
// earlier P V (two tiles: all of them; one tile: all but the last) are done.
// Few CTAs split the keys over a cluster of up to eight and join their parts
// through distributed shared memory in rank order.
#include <cuda.h>
#include <cuda_runtime.h>

#include "act16.cuh"
#include "cross_attention.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace rg {
namespace {

template <int D>
struct TileShape {
    static constexpr int NT = D == 256 ? 1 : 2;     // query tiles of a CTA
    static constexpr int NS = D == 256 ? 2 : 1;     // S buffers of a tile
    static constexpr int BKV = D == 256 ? 64 : 128;  // keys of a block
    static constexpr int QB = D < 64 ? 1 : D / 64;  // 64-column boxes of a row
    static constexpr int Q_BYTES = 128 * QB * 128;
    static constexpr int KV_BYTES = BKV * QB * 128;
    static constexpr int ST = 2;  // stages of K, and of V
    static constexpr int LOAD = NT * Q_BYTES + 2 * ST * KV_BYTES;
    static constexpr int PART = NT * D * 512;  // a CTA's fp32 outputs, when keys are split
    static constexpr int RING = LOAD > PART ? LOAD : PART;
    static constexpr int SMEM = RING + 2 * NT * 512 + 1024 + 256;
    static constexpr uint32_t S_COL(int t, int b) { return (t * NS + b) * BKV; }
    static constexpr uint32_t O_COL(int t) { return NT * NS * BKV + t * D; }
    static constexpr uint32_t TMEM_COLS = NT * NS * BKV + NT * D <= 256 ? 256 : 512;
    static constexpr int THREADS = 128 + 128 * NT;
    static_assert(NT * NS * BKV + NT * D <= 512 && SMEM <= 232448, "on-chip memory");
};

// registers of the two-tile kernel: 128 * 80 + 256 * 208 <= 384 * 168
constexpr int kControlRegs = 80, kSoftmaxRegs = 208;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

template <int D, bool F16>
__global__ void __launch_bounds__(TileShape<D>::THREADS, 1)
    cross_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, CrossParams p, int split, int qtiles) {
    using S = TileShape<D>;
    constexpr int NT = S::NT, NS = S::NS, BKV = S::BKV, QB = S::QB, ST = S::ST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                       // [NT][Q_BYTES]
    uint8_t* sK = sQ + NT * S::Q_BYTES;       // [ST][KV_BYTES]
    uint8_t* sV = sK + ST * S::KV_BYTES;      // [ST][KV_BYTES]
    float* sM = reinterpret_cast<float*>(smem + S::RING);  // [NT][128] maximum, then [NT][128] sum
    float* sL = sM + NT * 128;
    uint64_t* qfull = reinterpret_cast<uint64_t*>(sL + NT * 128);
    uint64_t* kfull = qfull + 1;
    uint64_t* kempty = kfull + ST;
    uint64_t* vfull = kempty + ST;
    uint64_t* vempty = vfull + ST;
    uint64_t* vfixed = vempty + ST;
    uint64_t* sfull = vfixed + 1;         // [NT][NS]
    uint64_t* pfull = sfull + NT * NS;    // [NT]
    uint64_t* ofull = pfull + NT;         // [NT]
    uint64_t* drain = ofull + NT;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    pdl_wait();  // the sequence table may come from the previous kernel
    const int rank = blockIdx.x % split, rest = blockIdx.x / split;
    const int s = rest / qtiles, h = blockIdx.y, hk = h / p.group;
    const int q0 = rest % qtiles * (128 * NT);
    CrossSeq c;
    if (!cross_seq(p, s, c, kStatusBadShape)) return;  // the same for every CTA of a cluster
    if (q0 >= c.nq) return;
    const int nt = min(NT, (c.nq - q0 + 127) / 128);
    const int blocks = (c.nk + BKV - 1) / BKV;
    // this CTA's share of the key blocks
    const int b0 = static_cast<int>(static_cast<int64_t>(blocks) * rank / split);
    const int nb = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / split) - b0;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(qfull, 1);
        for (int i = 0; i < ST; ++i) {
            mbar_init(&kfull[i], 1);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 1);
            mbar_init(&vempty[i], 1);
        }
        mbar_init(vfixed, 1);
        for (int i = 0; i < NT * NS; ++i) mbar_init(&sfull[i], 1);
        for (int t = 0; t < NT; ++t) {
            mbar_init(&pfull[t], 4);  // one arrival per softmax warp
            mbar_init(&ofull[t], 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, S::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();  // after the allocation: the next kernel's must not come between
    const uint32_t tmem = *tmem_slot;
    // keys of the last block, and whether the MMA step at its end has rows to clear
    const int tail = c.nk - (blocks - 1) * BKV;
    const bool last_here = nb > 0 && b0 + nb == blocks;
    const bool clear = last_here && (tail & 15) != 0;

    if (warp < 4) {
        if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == 0 && nb > 0) {
            // ---------------- TMA producer ----------------
            int ki = 0, vi = 0;  // blocks loaded
            if (elect_one()) {
                mbar_arrive_expect_tx(qfull, nt * S::Q_BYTES);
                for (int t = 0; t < nt; ++t)
                    for (int b = 0; b < QB; ++b)
                        tma_load_2d(sQ + t * S::Q_BYTES + b * 16384, &tmQ, qfull, h * D + b * 64, c.q0 + q0 + 128 * t);
            }
            __syncwarp();
            for (int i = 0; i < nb; ++i) {
                const int st = i % ST, row = c.k0 + (b0 + i) * BKV;
                const uint32_t ph = (i / ST) & 1;
                if (!mbar_wait_warp(&kempty[st], ph ^ 1, p.status, abort_flag)) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&kfull[st], S::KV_BYTES);
                    for (int b = 0; b < QB; ++b)
                        tma_load_2d(sK + st * S::KV_BYTES + b * BKV * 128, &tmK, &kfull[st], hk * D + b * 64, row);
                }
                __syncwarp();
                ki = i + 1;
                if (!mbar_wait_warp(&vempty[st], ph ^ 1, p.status, abort_flag)) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&vfull[st], S::KV_BYTES);
                    for (int b = 0; b < QB; ++b)
                        tma_load_2d(sV + st * S::KV_BYTES + b * BKV * 128, &tmV, &vfull[st], hk * D + b * 64, row);
                }
                __syncwarp();
                vi = i + 1;
            }
            if (clear && vi == nb) {
                const int st = (nb - 1) % ST;
                if (mbar_wait_warp(&vfull[st], ((nb - 1) / ST) & 1, p.status, abort_flag)) {
                    const int rows = 16 - (tail & 15);
                    for (int e = lane; e < rows * QB * 8; e += 32) {
                        const int b = e / (rows * 8), r = tail + e / 8 % rows;
                        *reinterpret_cast<uint4*>(sV + st * S::KV_BYTES + b * BKV * 128 + r * 128 + (e & 7) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(vfixed);
                }
            }
            // every load issued has landed before the CTA may exit
            mbar_drain(qfull, 0);
            for (int i = ki > ST ? ki - ST : 0; i < ki; ++i) mbar_drain(&kfull[i % ST], (i / ST) & 1);
            for (int i = vi > ST ? vi - ST : 0; i < vi; ++i) mbar_drain(&vfull[i % ST], (i / ST) & 1);
        } else if (warp == 1 && nb > 0) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t fmt = F16 ? 0u : 1u;
            constexpr uint32_t idS = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(BKV >> 3) << 17) |
                                     ((uint32_t)(128 >> 4) << 24);
            constexpr uint32_t idO = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                                     ((uint32_t)(128 >> 4) << 24);
            const uint64_t qd = sdesc_k128(smem_u32(sQ)), kd = sdesc_k128(smem_u32(sK));
            const uint64_t vd = sdesc_mn128(smem_u32(sV), BKV * 128);
            bool issued = false;
            auto qk = [&](int t, int i) {  // S of block i
                if (elect_one()) {
                    const uint32_t d = tmem + S::S_COL(t, i % NS);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_bf16(d, qd + (t * S::Q_BYTES + (ks >> 2) * 16384 + (ks & 3) * 32) / 16,
                                  kd + (i % ST * S::KV_BYTES + (ks >> 2) * BKV * 128 + (ks & 3) * 32) / 16, idS, ks > 0);
                    umma_commit(&sfull[t * NS + i % NS]);
                }
                __syncwarp();
                issued = true;
            };
            auto pv = [&](int t, int i, bool commit) {  // O += P V of block i
                const int steps = last_here && i + 1 == nb ? (tail + 15) / 16 : BKV / 16;
                if (elect_one()) {
                    const uint32_t d = tmem + S::O_COL(t), a = tmem + S::S_COL(t, i % NS);
#pragma unroll
                    for (int kk = 0; kk < BKV / 16; ++kk)
                        if (kk < steps)
                            umma_f16_ts(d, a + kk * 8, vd + (i % ST * S::KV_BYTES + kk * 2048) / 16, idO, (i | kk) != 0);
                    if (commit) umma_commit(&ofull[t]);
                }
                __syncwarp();
            };
            auto v_ready = [&](int i) -> bool {
                return mbar_wait_warp(&vfull[i % ST], (i / ST) & 1, p.status, abort_flag) &&
                       (!clear || i + 1 < nb || mbar_wait_warp(vfixed, 0, p.status, abort_flag));
            };
            auto commit_to = [&](uint64_t* bar) {
                if (elect_one()) umma_commit(bar);
                __syncwarp();
            };
            bool ok = mbar_wait_warp(qfull, 0, p.status, abort_flag) &&
                      mbar_wait_warp(&kfull[0], 0, p.status, abort_flag);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < nt; ++t) qk(t, 0);
                commit_to(&kempty[0]);
            }
            for (int i = 0; i < nb && ok; ++i) {
                const bool more = i + 1 < nb;
                if (NS == 2 && more) {  // the next block's S runs under this one's softmax
                    ok = mbar_wait_warp(&kfull[(i + 1) % ST], ((i + 1) / ST) & 1, p.status, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    qk(0, i + 1);
                    commit_to(&kempty[(i + 1) % ST]);
                }
                for (int t = 0; t < nt; ++t) {
                    ok = mbar_wait_warp(&pfull[t], i & 1, p.status, abort_flag) && (t > 0 || v_ready(i));
                    if (!ok) break;
                    tc_fence_after();
                    pv(t, i, NS == 2 || !more);
                    if (NS == 1 && more) {
                        if (t == 0 && !mbar_wait_warp(&kfull[(i + 1) % ST], ((i + 1) / ST) & 1, p.status, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        qk(t, i + 1);
                    }
                }
                if (!ok) break;
                commit_to(&vempty[i % ST]);
                if (NS == 1 && more) commit_to(&kempty[(i + 1) % ST]);
            }
            if (issued) {
                commit_to(drain);
                mbar_drain(drain, 0);
            }
        }
        // The control warps gave registers up: nothing is shared with the softmax
        // warps' code from here on but the barriers.
        __syncwarp();
        if (split > 1) {
            __syncthreads();
            cluster_sync();
            cluster_sync();
        }
        tc_fence_before();
        __syncthreads();
        if (warp == 2) {
            tc_fence_after();
            tmem_dealloc(tmem, S::TMEM_COLS);
        }
    } else {
        // ---------------- softmax, then the output ----------------
        float m = -INFINITY, l = 0.f;  // this row's maximum (exp2 domain) and sum
        const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        bool done = true;
        if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        if (t < nt) {
            const float scale = p.scale_log2;
            const uint32_t tO = tmem + S::O_COL(t) + lane_addr;
            for (int i = 0; i < nb; ++i) {
                const uint32_t tS = tmem + S::S_COL(t, i % NS) + lane_addr;
                done = mbar_wait_warp(&sfull[t * NS + i % NS], (i / NS) & 1, p.status, abort_flag);
                if (!done) break;
                tc_fence_after();
                uint32_t x[BKV];
#pragma unroll
                for (int j = 0; j < BKV; j += 32) tmem_ld32(tS + j, *reinterpret_cast<uint32_t(*)[32]>(&x[j]));
                tmem_ld_wait();
                if (last_here && i + 1 == nb && tail < BKV) {  // keys past the end
#pragma unroll
                    for (int j = 0; j < BKV; ++j)
                        if (j >= tail) x[j] = 0xff800000u;
                }
                float pm[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pm[j] = __uint_as_float(x[j]);
#pragma unroll
                for (int j = 8; j < BKV; j += 2)
                    pm[(j >> 1) & 7] = max3(pm[(j >> 1) & 7], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
                const float mx =
                    max3(max3(pm[0], pm[1], pm[2]), max3(pm[3], pm[4], pm[5]), fmaxf(pm[6], pm[7])) * scale;
                // The maximum in use stays until a block's is more than 8 above it:
                // P is at most 2^8, O is rescaled rarely, and the division by the sum
                // cancels it.
                const float now = mx > m + 8.0f ? mx : m;
                const float off = now == -INFINITY ? 0.f : -now;
                const float alpha = exp2_approx(m + off);
                m = now;
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    if (NS == 2) {
                        done = mbar_wait_warp(&ofull[t], (i - 1) & 1, p.status, abort_flag);
                        if (!done) break;
                        tc_fence_after();
                    }
#pragma unroll
                    for (int j = 0; j < D; j += 16) {
                        uint32_t o[16];
                        tmem_ld16(tO + j, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st16(tO + j, o);
                    }
                }
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < BKV; j += 32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float a = exp2_approx(fmaf(__uint_as_float(x[j + 2 * e]), scale, off));
                        const float b = exp2_approx(fmaf(__uint_as_float(x[j + 2 * e + 1]), scale, off));
                        ls[e & 3] += a + b;
                        // rounded to the 16 bits of V for the product, by at most half a step
                        pk[e] = pack2<F16>(a, b);
                    }
                    tmem_st16(tS + j / 2, pk);
                }
                l = l * alpha + ((ls[0] + ls[1]) + (ls[2] + ls[3]));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[t]);
            }
            // The last P V.  With two S buffers every P V is a phase of the barrier, and
            // the last S says no more than that the last but two are over: a wait can
            // tell two neighbouring phases apart, not three.
            if (NS == 2 && nb > 1) done = done && mbar_wait_warp(&ofull[t], nb & 1, p.status, abort_flag);
            if (nb > 0) done = done && mbar_wait_warp(&ofull[t], NS == 2 ? (nb - 1) & 1 : 0, p.status, abort_flag);
            tc_fence_after();
        }
        const int row = q0 + t * 128 + r;
        const bool stored = t < nt && done && row < c.nq;
        uint16_t* out = p.out + static_cast<int64_t>(c.q0 + row) * p.ldo + h * D;
        if (split == 1) {
            if (t < nt && done) {
                const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays
    #pragma unroll
                for (int j = 0; j < D; j += 16) {
                    uint32_t o[16];
                    if (nb > 0) {
                        tmem_ld16(tmem + S::O_COL(t) + lane_addr + j, o);
                        tmem_ld_wait();
                    } else {
    #pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = 0u;
                    }
                    if (stored) {
    #pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            uint4 u;
                            u.x = pack2<F16>(__uint_as_float(o[8 * v + 0]) * inv, __uint_as_float(o[8 * v + 1]) * inv);
                            u.y = pack2<F16>(__uint_as_float(o[8 * v + 2]) * inv, __uint_as_float(o[8 * v + 3]) * inv);
                            u.z = pack2<F16>(__uint_as_float(o[8 * v + 4]) * inv, __uint_as_float(o[8 * v + 5]) * inv);
                            u.w = pack2<F16>(__uint_as_float(o[8 * v + 6]) * inv, __uint_as_float(o[8 * v + 7]) * inv);
                            *reinterpret_cast<uint4*>(out + j + v * 8) = u;
                        }
                    }
                }
            }
        } else {
            // parts [NT][D][128] take the stages' place
            __syncthreads();
            float* part = reinterpret_cast<float*>(smem);
            if (t < nt) {
                sM[t * 128 + r] = m;
                sL[t * 128 + r] = l;
    #pragma unroll
                for (int j = 0; j < D; j += 16) {
                    uint32_t o[16];
                    if (nb > 0 && done) {
                        tmem_ld16(tmem + S::O_COL(t) + lane_addr + j, o);
                        tmem_ld_wait();
                    } else {
    #pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = 0u;
                    }
    #pragma unroll
                    for (int e = 0; e < 16; ++e) part[(t * D + j + e) * 128 + r] = __uint_as_float(o[e]);
                }
            }
            cluster_sync();
            if (stored) {
                // this rank's share of the head: columns [rank D / split, (rank + 1) D / split)
                float w[8], top = -INFINITY, sum = 0.f;
    #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    w[k] = k < split ? ld_shared_cluster(mapa_shared(smem_u32(sM + t * 128 + r), k)) : -INFINITY;
                    top = fmaxf(top, w[k]);
                }
    #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    w[k] = w[k] == -INFINITY ? 0.f : exp2_approx(w[k] - top);
                    if (k < split) sum += w[k] * ld_shared_cluster(mapa_shared(smem_u32(sL + t * 128 + r), k));
                }
                const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
                for (int j = rank * (D / split); j < (rank + 1) * (D / split); j += 8) {
                    float v[8];
    #pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = 0.f;
    #pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k < split && w[k] != 0.f)
                                v[e] += w[k] * ld_shared_cluster(mapa_shared(smem_u32(part + (t * D + j + e) * 128 + r), k));
                        v[e] *= inv;
                    }
                    *reinterpret_cast<uint4*>(out + j) = make_uint4(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]),
                                                                    pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7]));
                }
            }
            cluster_sync();  // a CTA's part is read until here
        }
        tc_fence_before();
        __syncthreads();
    }
}

template <int D, bool F16>
cudaError_t launch_tiles(const CrossParams& p, int num_sms, cudaStream_t st) {
    using S = TileShape<D>;
    auto kern = cross_tiles_kernel<D, F16>;
    static unsigned configured = 0;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 32 || !(__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & (1u << dev))) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 32) __atomic_fetch_or(&configured, 1u << dev, __ATOMIC_RELEASE);
    }
    CUtensorMap tq, tk, tv;
    if (!make_rows_tmap(&tq, p.q, p.f16, p.Tq, static_cast<uint64_t>(p.heads) * D, p.ldq, 128) ||
        !make_rows_tmap(&tk, p.k, p.f16, p.Tk, static_cast<uint64_t>(p.kv_heads) * D, p.ldk, S::BKV) ||
        !make_rows_tmap(&tv, p.v, p.f16, p.Tk, static_cast<uint64_t>(p.kv_heads) * D, p.ldv, S::BKV))
        return cudaErrorInvalidValue;
    const int qtiles = (p.max_q + 128 * S::NT - 1) / (128 * S::NT);
    const int64_t ctas = static_cast<int64_t>(p.nseq) * qtiles * p.heads;
    const int blocks = (p.max_kv + S::BKV - 1) / S::BKV;
    // keys are split over up to eight CTAs (of at least eight columns each in
    // the join) while these find room on the SMs and keep two blocks
    int split = 1;
    while (split < 8 && split * 8 < D && 2 * split * ctas <= num_sms && 4 * split <= blocks) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.nseq * qtiles * split, p.heads);
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
    return cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, p, split, qtiles);
}

}  // namespace

cudaError_t launch_cross_tiles(const CrossParams& p, int head_dim, int num_sms, cudaStream_t st) {
#define RG_CROSS_TILES(DD)                                        \
    if (head_dim == DD)                                           \
        return p.f16 ? launch_tiles<DD, true>(p, num_sms, st) : launch_tiles<DD, false>(p, num_sms, st);
    RG_CROSS_TILES(32)
    RG_CROSS_TILES(64)
    RG_CROSS_TILES(128)
    RG_CROSS_TILES(256)
#undef RG_CROSS_TILES
    return cudaErrorInvalidValue;
}

cudaError_t launch_cross(const CrossParams& p, int head_dim, int num_sms, cudaStream_t st) {
    const int64_t rows = static_cast<int64_t>(p.max_q) * p.group;
    if (rows <= 64 && (rows + 15) / 16 * p.kv_heads <= 65535) return launch_cross_rows(p, head_dim, num_sms, st);
    return launch_cross_tiles(p, head_dim, num_sms, st);
}

}  // namespace rg
