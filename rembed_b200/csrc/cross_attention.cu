// cross_attention.cu - cross attention on the 5th-generation tensor cores:
// tiles of 128 query rows of one (sequence, query head) against blocks of BKV
// keys, one pass with the running maximum and sum of the softmax.
//
// A CTA starts on the item of NT tiles (head dims up to 128: two, 384 threads;
// 256: one, 256 threads) of its block index and goes on with those of CTAs that
// have not started yet, taken over through cluster launch control: the next
// item's loads and first products run under the last softmax and the output of
// the one before, and the order of the hardware's scheduler evens the load out
// (8 x 2048 queries over 4096 keys, 12 heads x 64: 305 us in a fixed round of
// items, 275 in a CTA for each, 262 so).  Roles:
//   warp 0     takes items over, once the one before is all loaded (taken at its
//              start they would wait behind it while other SMs idle); TMA
//              producer of an item's query tiles, and of K and V blocks through
//              two stages each.  In a text's last block the rows of V behind its
//              end that share a 16-key MMA step with it are overwritten with
//              zeros (they may hold anything: 0 * NaN would reach the output);
//   warp 1     MMA issuer: S = Q K^T into tensor memory, O += P V with P read
//              from tensor memory, where it takes the place of its S (up to
//              head dim 128 in two halves, the first under the exponentials of
//              the second);
//   warp 2     TMEM allocator;
//   warps 4..  softmax, four warps a tile, thread = query row = TMEM lane.
// With two tiles the softmax of one runs under the MMAs of the other; the one
// tile of head dim 256 has two S buffers instead.  The tensor core finishes a
// thread's MMAs in order, so a block's S being ready implies that the tile's
// earlier P V (two tiles: all of them; one tile: all but the last) are done.
// A wait tells only two neighbouring phases of its barrier apart, so none may
// run ahead of its waiter by two: with two S buffers the softmax can be a whole
// block ahead of the issuer, and P and O have a barrier for each buffer.
// Few items split the keys over a cluster of up to eight CTAs and join their
// parts through distributed shared memory in rank order.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "act16.cuh"
#include "clusters.cuh"
#include "cross_attention.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace rg {
namespace {

template <int D>
struct TileShape {
    static constexpr int NT = D == 256 ? 1 : 2;     // query tiles of an item
    static constexpr int NS = D == 256 ? 2 : 1;     // S buffers of a tile
    static constexpr int BKV = D == 256 ? 64 : 128;  // keys of a block
    static constexpr int QB = D < 64 ? 1 : D / 64;  // 64-column boxes of a row
    static constexpr int Q_BYTES = 128 * QB * 128;
    static constexpr int KV_BYTES = BKV * QB * 128;
    static constexpr int LOAD = NT * Q_BYTES + 4 * KV_BYTES;  // Q, two stages of K and of V
    static constexpr int PART = NT * D * 512;  // a CTA's fp32 outputs, when keys are split
    static constexpr int RING = LOAD > PART ? LOAD : PART;
    static constexpr int SMEM = RING + 2 * NT * 512 + 512 + 1024;
    static constexpr uint32_t S_COL(int t, int b) { return (t * NS + b) * BKV; }
    static constexpr uint32_t O_COL(int t) { return NT * NS * BKV + t * D; }
    static constexpr uint32_t TMEM_COLS = NT * NS * BKV + NT * D <= 256 ? 256 : 512;
    static constexpr int THREADS = 128 + 128 * NT;
    // keys whose P is handed over before the rest of their block
    static constexpr int CUT = D == 256 ? BKV : BKV / 2;
    // Which pair of how many takes its exponentials on the FMA pipe: the
    // transcendental unit alone needs as long as the tensor core at head dim 128
    // and twice as long at 64 (8 x 2048 queries over 4096 keys, none, one in
    // eight, in four, in two: head dim 128 381, 366, 368, 401 us; 64 261, 248,
    // 246, 272 us).
    static constexpr int FMA_EVERY = D == 256 ? 64 : (D == 128 ? 8 : 4);
    static_assert(NT * NS * BKV + NT * D <= 512 && SMEM <= 232448, "on-chip memory");
    static_assert(NS == 1 || (NT == 1 && CUT == BKV), "pfull is by the cut or by the buffer");
    // The clusters of a split wait for all of their CTAs, and each of these for
    // its tensor memory.  No other kernel that holds tensor memory while its own
    // cluster waits may share an SM with one, or two calls on two streams could
    // wait for each other: two tiles take the SM's registers (384 x 168 of 65536),
    // one tile its shared memory.
    static_assert(NT == 2 || SMEM > 160 * 1024, "a CTA has its SM to itself");
};

template <int N>
struct Const {
    static constexpr int value = N;
};

// registers of the two-tile kernel: 128 * 72 + 256 * 216 = 384 * 168
constexpr int kControlRegs = 72, kSoftmaxRegs = 216;

// 2^x of a pair on the FMA pipe: n = round(x) by the magic constant 1.5 * 2^23,
// 2^f on [-1/2, 1/2] by a quartic fitted here for least relative error (2.7e-6
// in fp32), n added to the exponent.  Clamped at 2^-125, which is nothing beside
// a sum of at least one: a row's maximum is its reference or up to 2^8 above.  A
// row without such a maximum comes out by row_weight, and what it has gathered
// counts 0 times once it finds one; a row with a NaN or +infinity is NaN already.
__device__ __forceinline__ void exp2_fma(float& a, float& b) {
    const uint64_t x = pair_of(fmaxf(a, -125.0f), fmaxf(b, -125.0f));
    const uint64_t magic = pair_of(12582912.0f, 12582912.0f);
    const uint64_t t = add_pair(x, magic);
    const uint64_t f = add_pair(x, fma_pair(t, pair_of(-1.0f, -1.0f), magic));
    uint64_t y = fma_pair(pair_of(0.009570102207362652f, 0.009570102207362652f), f,
                          pair_of(0.05591785907745361f, 0.05591785907745361f));
    y = fma_pair(y, f, pair_of(0.240247443318367f, 0.240247443318367f));
    y = fma_pair(y, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
    y = fma_pair(y, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
    float ta, tb;
    split_pair(y, a, b);
    split_pair(t, ta, tb);
    a = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23));
    b = __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23));
}
// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// One item: up to NT tiles of one (sequence, query head), and this CTA's blocks
// of the sequence's keys.
struct Work {
    int h, row, rows;  // query head, -1 for no more items; first row of q and out; rows from there to the sequence's end
    int nt;            // tiles with rows, 0 for an item without
    int k0, nb;        // first row of k and v, blocks of keys
    int tail;          // keys of the last of the nb blocks
    int clear;         // it ends within a 16-key step
    int keys;          // the sequence has keys
};

template <int D>
__device__ __forceinline__ Work work_of(const CrossParams& p, int item, int qtiles, int rank, int split, bool report) {
    using S = TileShape<D>;
    Work w = {};
    const int qt = item % qtiles, sh = item / qtiles;
    w.h = sh % p.heads;
    CrossSeq c;
    if (!cross_seq(p, sh / p.heads, c, report ? kStatusBadShape : 0)) return w;
    const int q0 = qt * (128 * S::NT);
    w.row = c.q0 + q0;
    w.rows = c.nq - q0;
    if (w.rows <= 0) return w;
    w.nt = min(S::NT, (w.rows + 127) / 128);
    const int blocks = (c.nk + S::BKV - 1) / S::BKV;
    const int b0 = static_cast<int>(static_cast<int64_t>(blocks) * rank / split);
    const int b1 = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / split);
    w.k0 = c.k0 + b0 * S::BKV;
    w.nb = b1 - b0;
    w.tail = b1 == blocks ? c.nk - (blocks - 1) * S::BKV : S::BKV;
    w.clear = w.nb > 0 && (w.tail & 15) != 0;
    w.keys = c.nk > 0;
    return w;
}

template <int D, bool F16>
__global__ void __launch_bounds__(TileShape<D>::THREADS, 1)
    cross_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, CrossParams p, int split, int qtiles) {
    using S = TileShape<D>;
    constexpr int NT = S::NT, NS = S::NS, BKV = S::BKV, QB = S::QB;
    constexpr int STEPS = BKV / 16, CUT = S::CUT / 16;  // MMA steps of a block, and before the cut
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                    // [NT][Q_BYTES]
    uint8_t* sK = sQ + NT * S::Q_BYTES;    // [2][KV_BYTES]
    uint8_t* sV = sK + 2 * S::KV_BYTES;    // [2][KV_BYTES]
    float* sM = reinterpret_cast<float*>(smem + S::RING);  // [NT][128] maximum, then [NT][128] sum
    float* sL = sM + NT * 128;
    uint64_t* qfull = reinterpret_cast<uint64_t*>(sL + NT * 128);
    uint64_t* qempty = qfull + 1;
    uint64_t* kfull = qempty + 1;         // [2]
    uint64_t* kempty = kfull + 2;         // [2]
    uint64_t* vfull = kempty + 2;         // [2]
    uint64_t* vempty = vfull + 2;         // [2]
    uint64_t* vfixed = vempty + 2;        // [2]: of a stage, so that none runs ahead of its reader
    uint64_t* sfull = vfixed + 2;         // [NT][NS]
    uint64_t* pfull = sfull + NT * NS;    // [NT][2]: before and after the cut, or of each S buffer
    uint64_t* ofull = pfull + NT * 2;     // [NT][NS]
    uint64_t* drain = ofull + NT * NS;
    uint64_t* taken = drain + 1;          // a response has come
    uint64_t* ifull = taken + 1;          // [2]: an item is there
    uint64_t* iempty = ifull + 2;         // [2]: every warp has read it
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(iempty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Work* sWork = reinterpret_cast<Work*>(tmem_slot + 2);  // [2]
    uint8_t* response = smem + S::SMEM - 1024 - 16;
    static_assert(2 * sizeof(Work) <= 128, "the barriers' 512 bytes");

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(qfull, 1);
        mbar_init(taken, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ifull[i], 1);
            mbar_init(&iempty[i], 1 + 4 * NT);  // issuer, softmax warps
        }
        mbar_init(qempty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&kfull[i], 1);
            mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], 1);
            mbar_init(&vempty[i], 1);
            mbar_init(&vfixed[i], 1);
        }
        for (int i = 0; i < NT * NS; ++i) mbar_init(&sfull[i], 1);
        for (int i = 0; i < NT * 2; ++i) mbar_init(&pfull[i], 4);  // one arrival per softmax warp
        for (int i = 0; i < NT * NS; ++i) mbar_init(&ofull[i], 1);
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
    pdl_wait();
    const uint32_t tmem = *tmem_slot;
    const int rank = blockIdx.x % split;
    const int first = blockIdx.x / split;
    // the k-th item of this CTA, as the producer passes it on
    auto item_at = [&](uint32_t k) -> Work {
        Work w = {};
        w.h = -1;
        // a warp without rows in an item waits here for as long as the others work
        // on it; each of their waits has its own limit and ends this one too
        if (!mbar_wait_warp(&ifull[k & 1], (k >> 1) & 1, p.status, abort_flag, 64 * kWaitLimitCycles)) return w;
        w = sWork[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&iempty[k & 1]);
        return w;
    };

    if (warp < 4) {
        if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == 0) {
            // ---------------- TMA producer ----------------
            uint32_t qn = 0, kn = 0, vn = 0;  // items, blocks of K and blocks of V loaded
            bool ok = true;
            // pass the k-th item on, as others read it from shared memory
            auto pass = [&](uint32_t k, const Work& w) -> bool {
                if (!mbar_wait_warp(&iempty[k & 1], ((k >> 1) & 1) ^ 1, p.status, abort_flag)) return false;
                if (lane == 0) {
                    sWork[k & 1] = w;
                    mbar_arrive(&ifull[k & 1]);
                }
                __syncwarp();
                return true;
            };
            // take one over: the k-th question; -1 if there is none
            auto take = [&](uint32_t k) -> int {
                if (elect_one()) {
                    mbar_arrive_expect_tx(taken, 16);
                    clc_try_cancel(response, taken);
                }
                __syncwarp();
                if (!mbar_wait_warp(taken, k & 1, p.status, abort_flag)) {
                    mbar_drain(taken, k & 1);  // the response may still be on its way
                    return -1;
                }
                const int item = clc_taken(response);
                fence_proxy_async_smem();  // read before the next response is written
                return item;
            };
            int item = first;
            for (uint32_t k = 0; ok; ++k) {
                Work w = {};
                w.h = -1;
                if (item >= 0) w = work_of<D>(p, item, qtiles, rank, split, lane == 0);
                ok = pass(k, w);
                if (w.h < 0 || !ok) break;
                if (w.nt == 0 || w.nb == 0) {
                    item = split > 1 ? -1 : take(k);
                    continue;
                }
                const int hk = w.h / p.group;
                ok = mbar_wait_warp(qempty, (qn & 1) ^ 1, p.status, abort_flag);
                if (!ok) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(qfull, w.nt * S::Q_BYTES);
                    for (int t = 0; t < w.nt; ++t)
                        for (int b = 0; b < QB; ++b)
                            tma_load_2d(sQ + t * S::Q_BYTES + b * 16384, &tmQ, qfull, w.h * D + b * 64, w.row + 128 * t);
                }
                __syncwarp();
                ++qn;
                for (int i = 0; i < w.nb; ++i) {
                    const int st = kn & 1, row = w.k0 + i * BKV;
                    const uint32_t ph = (kn >> 1) & 1;
                    ok = mbar_wait_warp(&kempty[st], ph ^ 1, p.status, abort_flag);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(&kfull[st], S::KV_BYTES);
                        for (int b = 0; b < QB; ++b)
                            tma_load_2d(sK + st * S::KV_BYTES + b * BKV * 128, &tmK, &kfull[st], hk * D + b * 64, row);
                    }
                    __syncwarp();
                    ++kn;
                    ok = mbar_wait_warp(&vempty[st], ph ^ 1, p.status, abort_flag);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(&vfull[st], S::KV_BYTES);
                        for (int b = 0; b < QB; ++b)
                            tma_load_2d(sV + st * S::KV_BYTES + b * BKV * 128, &tmV, &vfull[st], hk * D + b * 64, row);
                    }
                    __syncwarp();
                    ++vn;
                }
                if (ok && w.clear) {
                    const int st = (vn - 1) & 1;
                    ok = mbar_wait_warp(&vfull[st], ((vn - 1) >> 1) & 1, p.status, abort_flag);
                    if (!ok) break;
                    const int rows = 16 - (w.tail & 15);
                    for (int e = lane; e < rows * QB * 8; e += 32) {
                        const int b = e / (rows * 8), r = w.tail + e / 8 % rows;
                        *reinterpret_cast<uint4*>(sV + st * S::KV_BYTES + b * BKV * 128 + r * 128 + (e & 7) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&vfixed[st]);
                }
                if (ok) item = split > 1 ? -1 : take(k);
            }
            // every load issued has landed before the CTA may exit
            if (qn > 0) mbar_drain(qfull, (qn - 1) & 1);
            for (uint32_t i = kn > 2 ? kn - 2 : 0; i < kn; ++i) mbar_drain(&kfull[i & 1], (i >> 1) & 1);
            for (uint32_t i = vn > 2 ? vn - 2 : 0; i < vn; ++i) mbar_drain(&vfull[i & 1], (i >> 1) & 1);
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t fmt = F16 ? 0u : 1u;
            constexpr uint32_t idS = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(BKV >> 3) << 17) |
                                     ((uint32_t)(128 >> 4) << 24);
            constexpr uint32_t idO = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                                     ((uint32_t)(128 >> 4) << 24);
            // The operands of a tcgen05.mma come from uniform registers: stages and
            // tiles are compile-time constants here, so that descriptors are a
            // base plus a constant and nothing is moved over for each of them (a
            // 128 x 128 x 16 product takes the tensor core 64 cycles).
            const uint32_t qd = static_cast<uint32_t>(sdesc_k128(smem_u32(sQ)));
            const uint32_t kd = static_cast<uint32_t>(sdesc_k128(smem_u32(sK)));
            const uint32_t vd = static_cast<uint32_t>(sdesc_mn128(smem_u32(sV), BKV * 128));
            uint32_t qn = 0, n = 0;             // items and blocks so far
            uint32_t fixed[2] = {};             // cleared blocks of each stage so far
            uint32_t cn[NT] = {};               // blocks of each tile so far
            bool ok = true;
            auto commit_to = [&](uint64_t* bar) {
                if (elect_one()) umma_commit(bar);
                __syncwarp();
            };
            auto qk = [&](auto tc, auto stc) {  // S of a block in stage st
                constexpr int t = decltype(tc)::value, st = decltype(stc)::value;
                constexpr int buf = NS == 2 ? st : 0;
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_f16_ss(tmem + S::S_COL(t, buf), qd + (t * S::Q_BYTES + (ks >> 2) * 16384 + (ks & 3) * 32) / 16,
                                    kd + (st * S::KV_BYTES + (ks >> 2) * BKV * 128 + (ks & 3) * 32) / 16, idS, ks > 0);
                    umma_commit(&sfull[t * NS + buf]);
                }
                __syncwarp();
            };
            // O += P V (O starts as zeros), the steps before the cut as soon as their P is there
            auto pv = [&](auto tc, auto stc, int steps, bool commit) -> bool {
                constexpr int t = decltype(tc)::value, st = decltype(stc)::value;
                constexpr int buf = NS == 2 ? st : 0;
                const uint32_t ph = (cn[t]++ / NS) & 1;
                auto mma = [&](int kk) {
                    umma_f16_ts(tmem + S::O_COL(t), tmem + S::S_COL(t, buf) + kk * 8, vd + (st * S::KV_BYTES + kk * 2048) / 16,
                                idO, 1);
                };
                if (!mbar_wait_warp(&pfull[2 * t + buf], ph, p.status, abort_flag)) return false;
                tc_fence_after();
                if (elect_one()) {
                    if (steps >= CUT) {
#pragma unroll
                        for (int kk = 0; kk < CUT; ++kk) mma(kk);
                    } else {
                        for (int kk = 0; kk < steps; ++kk) mma(kk);
                    }
                    if (CUT == STEPS && commit) umma_commit(&ofull[t * NS + buf]);
                }
                __syncwarp();
                if constexpr (CUT < STEPS) {
                    if (!mbar_wait_warp(&pfull[2 * t + 1], ph, p.status, abort_flag)) return false;
                    tc_fence_after();
                    if (elect_one()) {
                        if (steps == STEPS) {
#pragma unroll
                            for (int kk = CUT; kk < STEPS; ++kk) mma(kk);
                        } else {
                            for (int kk = CUT; kk < steps; ++kk) mma(kk);
                        }
                        if (commit) umma_commit(&ofull[t * NS]);
                    }
                    __syncwarp();
                }
                return true;
            };
            for (uint32_t k = 0; ok; ++k) {
                const Work w = item_at(k);
                if (w.h < 0) break;
                if (w.nt == 0 || w.nb == 0) continue;
                // block i of the item, in stage st: its P V, and before (NS == 2) or
                // between the tiles' (NS == 1) the next block's S
                auto block = [&](int i, auto stc) -> bool {
                    constexpr int st = decltype(stc)::value;
                    constexpr Const<1 - st> next{};
                    const bool more = i + 1 < w.nb;
                    const uint32_t ph = (n >> 1) & 1, nph = ((n + 1) >> 1) & 1;
                    ++n;
                    const int steps = more ? STEPS : (w.tail + 15) / 16;
                    if (NS == 2 && more) {
                        if (!mbar_wait_warp(&kfull[1 - st], nph, p.status, abort_flag)) return false;
                        tc_fence_after();
                        qk(Const<0>{}, next);
                        commit_to(&kempty[1 - st]);
                        if (i + 2 == w.nb) commit_to(qempty);
                    }
                    if (!mbar_wait_warp(&vfull[st], ph, p.status, abort_flag)) return false;
                    if (w.clear && !more && !mbar_wait_warp(&vfixed[st], fixed[st]++ & 1, p.status, abort_flag))
                        return false;
                    if (!pv(Const<0>{}, stc, steps, NS == 2 || !more)) return false;
                    if (NS == 1 && more) {
                        if (!mbar_wait_warp(&kfull[1 - st], nph, p.status, abort_flag)) return false;
                        tc_fence_after();
                        qk(Const<0>{}, next);
                    }
                    if (NT == 2 && w.nt == 2) {
                        if (!pv(Const<NT - 1>{}, stc, steps, !more)) return false;
                        if (more) qk(Const<NT - 1>{}, next);
                    }
                    commit_to(&vempty[st]);
                    if (NS == 1 && more) {
                        commit_to(&kempty[1 - st]);
                        if (i + 2 == w.nb) commit_to(qempty);
                    }
                    return true;
                };
                auto begin = [&](auto stc) {
                    constexpr int st = decltype(stc)::value;
                    qk(Const<0>{}, stc);
                    if (NT == 2 && w.nt == 2) qk(Const<NT - 1>{}, stc);
                    commit_to(&kempty[st]);
                    if (w.nb == 1) commit_to(qempty);
                };
                ok = mbar_wait_warp(qfull, qn++ & 1, p.status, abort_flag) &&
                     mbar_wait_warp(&kfull[n & 1], (n >> 1) & 1, p.status, abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (n & 1) begin(Const<1>{});
                else begin(Const<0>{});
                for (int i = 0; i < w.nb && ok; ++i) ok = n & 1 ? block(i, Const<1>{}) : block(i, Const<0>{});
            }
            if (qn > 0) {
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
        if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t tO = tmem + S::O_COL(t) + lane_addr;
        const float scale = p.scale_log2;
        // rows of out on 32-byte boundaries: a thread stores whole sectors
        const bool sectors = (reinterpret_cast<uintptr_t>(p.out) & 31) == 0 && p.ldo % 16 == 0;
        uint32_t cn = 0, on = 0;        // blocks and outputs of this tile so far
        // this row's maximum (a score), its reference, and sum
        float m = -INFINITY, ref = -INFINITY, l = 0.f;
        Work w = {};  // split: still there for the join
        bool done = true;
        for (uint32_t k = 0; done; ++k) {
            const Work next = item_at(k);
            if (next.h < 0) break;
            w = next;
            if (t >= w.nt) continue;
            m = ref = -INFINITY;
            l = 0.f;
            if (w.nb > 0) {
                const uint32_t zero[16] = {};
#pragma unroll
                for (int j = 0; j < D; j += 16) tmem_st16(tO + j, zero);
            }
            for (int i = 0; i < w.nb; ++i, ++cn) {
                const int buf = NS == 2 ? cn & 1 : 0;
                const uint32_t tS = tmem + S::S_COL(t, buf) + lane_addr;
                done = mbar_wait_warp(&sfull[t * NS + buf], (cn / NS) & 1, p.status, abort_flag);
                if (!done) break;
                tc_fence_after();
                uint32_t x[BKV];
#pragma unroll
                for (int j = 0; j < BKV; j += 32) tmem_ld32(tS + j, *reinterpret_cast<uint32_t(*)[32]>(&x[j]));
                tmem_ld_wait();
                if (i + 1 == w.nb && w.tail < BKV) {  // keys past the end, by chunks
#pragma unroll
                    for (int j = 0; j < BKV; j += 32)
                        if (j + 32 > w.tail) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (j + e >= w.tail) x[j + e] = 0xff800000u;
                        }
                }
                float pm[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pm[j] = __uint_as_float(x[j]);
#pragma unroll
                for (int j = 8; j < BKV; j += 2)
                    pm[(j >> 1) & 7] = max3(pm[(j >> 1) & 7], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
                const float mx = max3(max3(pm[0], pm[1], pm[2]), max3(pm[3], pm[4], pm[5]), max3(pm[6], pm[7], pm[7]));
                // The maximum in use stays until a block's is more than 8 above it in
                // the exponent: P is at most 2^8 (fp16 2^15), O is rescaled rarely, and the
                // division by the sum cancels it.  A NaN or +infinity among the scores makes the
                // row NaN.
                const float mxr = reference<F16>(mx, scale);
                const bool up = mxr > ref + 8.0f;
                const float now = up ? mxr : ref;
                float off = mx < INFINITY ? -now : mx - mx;
                float alpha = ex2(ref + off);
                const bool far = fabsf(now) > kFar;
                if (__any_sync(0xffffffffu, alpha != 1.0f || far)) {
                    if (far) {  // hardly ever
                        far_maximum<F16>(mx, scale, m, ref, alpha);
                        if (mx < INFINITY) off = kLift<F16>;
                        if (m > -INFINITY) {
#pragma unroll
                            for (int j = 0; j < BKV; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) - m);
                        }
                    }
                    __syncwarp();
                    if (i > 0) {
                        if (NS == 2) {
                            done = mbar_wait_warp(&ofull[t * NS + (cn - 1) % NS], ((cn - 1) / NS) & 1, p.status, abort_flag);
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
                }
                if (!far) {
                    m = up ? mx : m;
                    ref = now;
                }
                const uint64_t scale2 = pair_of(scale, scale), off2 = pair_of(off, off);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < BKV; j += 32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float a, b;
                        split_pair(fma_pair(pair_of(__uint_as_float(x[j + 2 * e]), __uint_as_float(x[j + 2 * e + 1])), scale2,
                                            off2), a, b);
                        if (e % S::FMA_EVERY == S::FMA_EVERY - 1) {
                            exp2_fma(a, b);
                        } else {
                            a = ex2(a);
                            b = ex2(b);
                        }
                        sum2[e & 1] = add_pair(sum2[e & 1], pair_of(a, b));
                        // rounded to the 16 bits of V for the product, by at most half a step
                        pk[e] = pack2<F16>(a, b);
                    }
                    tmem_st16(tS + j / 2, pk);
                    if (j + 32 == S::CUT || j + 32 == BKV) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&pfull[2 * t + (NS == 2 ? buf : j + 32 > S::CUT)]);
                    }
                }
                float sa, sb;
                split_pair(add_pair(sum2[0], sum2[1]), sa, sb);
                l = l * alpha + (sa + sb);
            }
            if (!done) break;
            // the last P V (one S buffer: only it commits)
            if (w.nb > 0) {
                const uint32_t last = NS == 2 ? cn - 1 : on++;
                done = mbar_wait_warp(&ofull[t * NS + (NS == 2 ? last % NS : 0)], (last / NS) & 1, p.status, abort_flag);
            }
            if (!done) break;
            tc_fence_after();
            if (split == 1) {
                const float inv = row_weight(m, l, w.keys);
                uint16_t* out = p.out + static_cast<int64_t>(w.row + t * 128 + r) * p.ldo + w.h * D;
#pragma unroll
                for (int j = 0; j < D; j += 16) {
                    uint32_t o[16];
                    if (w.nb > 0) {
                        tmem_ld16(tO + j, o);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = 0u;
                    }
                    if (t * 128 + r < w.rows) {
                        uint32_t u[8];
#pragma unroll
                        for (int v = 0; v < 8; ++v)
                            u[v] = pack2<F16>(__uint_as_float(o[2 * v]) * inv, __uint_as_float(o[2 * v + 1]) * inv);
                        if (sectors) {
                            st_global_32(out + j, u);
                        } else {
                            *reinterpret_cast<uint4*>(out + j) = make_uint4(u[0], u[1], u[2], u[3]);
                            *reinterpret_cast<uint4*>(out + j + 8) = make_uint4(u[4], u[5], u[6], u[7]);
                        }
                    }
                }
            }
        }
        if (split > 1) {  // one item: its parts [NT][D][128] take the stages' place
            __syncthreads();
            float* part = reinterpret_cast<float*>(smem);
            if (t < w.nt) {
                sM[t * 128 + r] = m;
                sL[t * 128 + r] = l;
#pragma unroll
                for (int j = 0; j < D; j += 16) {
                    uint32_t o[16];
                    if (w.nb > 0 && done) {
                        tmem_ld16(tO + j, o);
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
            if (t < w.nt && done && t * 128 + r < w.rows) {
                // this rank's share of the head: columns [rank D / split, (rank + 1) D / split)
                float f[8], top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    f[k] = k < split ? ld_shared_cluster(mapa_shared(smem_u32(sM + t * 128 + r), k)) : -INFINITY;
                    top = fmaxf(top, f[k]);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    f[k] = f[k] == -INFINITY ? 0.f : ex2(reference_step<F16>(f[k], top, scale));
                    if (k < split) sum += f[k] * ld_shared_cluster(mapa_shared(smem_u32(sL + t * 128 + r), k));
                }
                const float inv = row_weight(top, sum, w.keys);
                uint16_t* out = p.out + static_cast<int64_t>(w.row + t * 128 + r) * p.ldo + w.h * D;
                for (int j = rank * (D / split); j < (rank + 1) * (D / split); j += 8) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = 0.f;
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k < split && f[k] != 0.f)
                                v[e] += f[k] * ld_shared_cluster(mapa_shared(smem_u32(part + (t * D + j + e) * 128 + r), k));
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
CrossPlan plan_tiles(const CrossParams& p, int num_sms) {
    using S = TileShape<D>;
    static ClusterCounts known = {};
    const int qtiles = (p.max_q + 128 * S::NT - 1) / (128 * S::NT);
    const int blocks = (p.max_kv + S::BKV - 1) / S::BKV;
    CrossPlan plan = {static_cast<int64_t>(p.nseq) * qtiles * p.heads, 1, cudaSuccess};
    // keys are split over up to eight CTAs (of at least eight columns each in
    // the join) while these all run at once and keep two blocks (one text of
    // 4096 keys, 16/8 heads x 128: 33 us over eight, two rounds of clusters; 28
    // over four)
    int fit = 0;
    plan.error = clusters_at_once(cross_tiles_kernel<D, F16>, S::THREADS, S::SMEM, 1, known, fit);
    for (int split = 2; split <= 8 && plan.error == cudaSuccess; split *= 2) {
        if (split * 8 > D || split * plan.ctas > num_sms || 2 * split > blocks) break;
        plan.error = clusters_at_once(cross_tiles_kernel<D, F16>, S::THREADS, S::SMEM, split, known, fit);
        if (plan.error != cudaSuccess || plan.ctas > fit) break;
        plan.split = split;
    }
    return plan;
}

template <int D, bool F16>
cudaError_t launch_tiles(const CrossParams& p, int split, cudaStream_t st) {
    using S = TileShape<D>;
    auto kern = cross_tiles_kernel<D, F16>;
    CUtensorMap tq, tk, tv;
    if (!make_rows_tmap(&tq, p.q, p.f16, p.Tq, static_cast<uint64_t>(p.heads) * D, p.ldq, 128) ||
        !make_rows_tmap(&tk, p.k, p.f16, p.Tk, static_cast<uint64_t>(p.kv_heads) * D, p.ldk, S::BKV) ||
        !make_rows_tmap(&tv, p.v, p.f16, p.Tk, static_cast<uint64_t>(p.kv_heads) * D, p.ldv, S::BKV))
        return cudaErrorInvalidValue;
    const int qtiles = (p.max_q + 128 * S::NT - 1) / (128 * S::NT);
    const int64_t items = static_cast<int64_t>(p.nseq) * qtiles * p.heads;
    if (items > 0x7fffffff / 16) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * split));
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

CrossPlan plan_cross_tiles(const CrossParams& p, int head_dim, int num_sms) {
#define RG_CROSS_TILES(DD)                                        \
    if (head_dim == DD)                                           \
        return p.f16 ? plan_tiles<DD, true>(p, num_sms) : plan_tiles<DD, false>(p, num_sms);
    RG_CROSS_TILES(32)
    RG_CROSS_TILES(64)
    RG_CROSS_TILES(128)
    RG_CROSS_TILES(256)
#undef RG_CROSS_TILES
    return {0, 1, cudaErrorInvalidValue};
}

cudaError_t launch_cross_tiles(const CrossParams& p, int head_dim, int split, cudaStream_t st) {
#define RG_CROSS_TILES(DD)                                        \
    if (head_dim == DD)                                           \
        return p.f16 ? launch_tiles<DD, true>(p, split, st) : launch_tiles<DD, false>(p, split, st);
    RG_CROSS_TILES(32)
    RG_CROSS_TILES(64)
    RG_CROSS_TILES(128)
    RG_CROSS_TILES(256)
#undef RG_CROSS_TILES
    return cudaErrorInvalidValue;
}

// The row kernel takes 16 rows of a key/value head to a CTA and reads K and V for
// each of them, the tile kernel up to 256 rows of a query head.  Each one's time
// is taken as a start and, for every round of its CTAs over the SMs, a constant
// and a time for each key that a CTA goes through: microseconds, fitted to calls
// of 1 to 4 texts of 512 and of 4096 keys with 4 to 256 tokens and to 64 texts
// of 300 keys (rows against tiles, 2 texts of 4096 keys, 3/1 heads x 256: 32
// tokens 23 and 25 us, 64 33 and 26, 128 51 and 27; 64 texts, 12/12 x 64: 32
// tokens 34 and 39 us, 48 45 and 39; 16/8 x 128: 16 tokens 41 and 51, 32 63 and
// 51).
cudaError_t launch_cross(const CrossParams& p, int head_dim, int num_sms, cudaStream_t st) {
    struct Cost {
        float rows, rows_key, start, tiles, tiles_key;
    };
    const Cost us = head_dim == 32    ? Cost{1.0f, 0.0050f, 1.2f, 2.0f, 0.0100f}
                    : head_dim == 64  ? Cost{2.5f, 0.0075f, 5.0f, 2.0f, 0.0100f}
                    : head_dim == 128 ? Cost{3.5f, 0.0125f, 7.0f, 2.0f, 0.0125f}
                                      : Cost{5.0f, 0.0172f, 7.0f, 2.0f, 0.0165f};
    const int64_t tiles = (static_cast<int64_t>(p.max_q) * p.group + 15) / 16 * p.kv_heads;
    const CrossPlan by_tiles = plan_cross_tiles(p, head_dim, num_sms);
    if (by_tiles.error != cudaSuccess) return by_tiles.error;
    if (tiles <= 65535) {
        const CrossPlan by_rows = plan_cross_rows(p, head_dim, num_sms);
        if (by_rows.error != cudaSuccess) return by_rows.error;
        auto rounds = [](const CrossPlan& plan, int room) {
            return std::max(1.0f, static_cast<float>(plan.ctas) * static_cast<float>(plan.split) / static_cast<float>(room));
        };
        auto keys = [&](const CrossPlan& plan) { return static_cast<float>(p.max_kv) / static_cast<float>(plan.split); };
        // at head dim 256 an SM holds one row CTA: a started round takes as long as a full one
        const float turns = head_dim == 256 ? std::ceil(rounds(by_rows, num_sms)) : rounds(by_rows, 2 * num_sms);
        const float rows = turns * (us.rows + us.rows_key * keys(by_rows));
        const float whole = us.start + rounds(by_tiles, num_sms) * (us.tiles + us.tiles_key * keys(by_tiles));
        if (rows <= whole) return launch_cross_rows(p, head_dim, by_rows.split, st);
    }
    return launch_cross_tiles(p, head_dim, by_tiles.split, st);
}

}  // namespace rg
