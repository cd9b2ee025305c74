// cross_attention_rows.cu - cross attention of few query rows: a decoder's
// single tokens over an encoder's keys and values.
//
// Rows are the (token, query head) pairs of one sequence that share a
// key/value head, 16 to a tile.  All such a call has to do is to read K and V
// once: per key and 16-bit head dim D it reads 4 D bytes and multiplies 2 x 16
// x D, a ratio that leaves the warp-level tensor instructions idle most of the
// time even with one row in sixteen filled.  So every warp runs on its own:
// it takes every 4th (x split) chunk of keys through its own ring of
// asynchronous copies and keeps running maximum, sum and output in registers;
// the warps' parts are joined at the end, across up to eight CTAs of a cluster
// through distributed shared memory, in a fixed order.  Keys past the end are
// zero-filled by the copies (nothing outside a sequence is read) and masked.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "act16.cuh"
#include "clusters.cuh"
#include "cross_attention.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace rg {
namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;

template <int D>
struct RowsShape {
    static constexpr int KEYS = D <= 64 ? 32 : 16;  // keys of a chunk
    // of chunks: room for three CTAs an SM (head dim 256: one); keys are split while
    // the parts fit two an SM
    static constexpr int STAGES = D == 32 ? 4 : 2;
    static constexpr int CHUNK = KEYS * D * 2;  // bytes of a chunk of K, and of V
    static constexpr int RING = STAGES * 2 * CHUNK;
    // at the end a warp's 16 x D fp32 outputs take its ring's place
    static_assert(RING >= kRows * D * 4, "a warp's outputs take its ring's place");
    // rings | maximum, sum, weight [kWarps][kRows] | maximum, sum of all [kRows]
    static constexpr int SMEM = kWarps * RING + (3 * kWarps + 2) * kRows * 4;
};

// Byte offset of 16-byte piece c of row r in a chunk, so that eight
// neighbouring rows' pieces fall on different banks.
template <int D>
__device__ __forceinline__ int piece(int r, int c) {
    if constexpr (D == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    else return r * D * 2 + (((c & ~7) | ((c ^ r) & 7)) << 4);
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, bool F16>
__global__ void __launch_bounds__(32 * kWarps) cross_rows_kernel(CrossParams p, int split) {
    using S = RowsShape<D>;
    constexpr int KEYS = S::KEYS, STAGES = S::STAGES, CHUNK = S::CHUNK, NT = KEYS / 8;
    pdl_trigger();
    pdl_wait();
    const int rank = blockIdx.x % split, s = blockIdx.x / split;
    const int hk = blockIdx.y % p.kv_heads, tile = blockIdx.y / p.kv_heads;
    CrossSeq c;
    if (!cross_seq(p, s, c, threadIdx.x == 0 ? kStatusBadShape : 0)) return;  // the same for every CTA of a cluster
    const int rows = min(kRows, c.nq * p.group - tile * kRows);
    if (rows <= 0) return;

    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* sM = reinterpret_cast<float*>(smem + kWarps * S::RING);  // [kWarps][kRows]
    float* sL = sM + kWarps * kRows;
    float* sW = sL + kWarps * kRows;  // [kWarps][kRows]
    float* sTop = sW + kWarps * kRows;
    float* sSum = sTop + kRows;
    const uint32_t ring = smem_u32(smem) + warp * S::RING;

    // this warp's chunks: step apart from its own number on
    const int chunks = (c.nk + KEYS - 1) / KEYS;
    const int step = split * kWarps, first = rank * kWarps + warp;
    const uint16_t* kbase = p.k + static_cast<int64_t>(c.k0) * p.ldk + hk * D;
    const uint16_t* vbase = p.v + static_cast<int64_t>(c.k0) * p.ldv + hk * D;
    auto load = [&](int chunk, int stage) {
        if (chunk < chunks) {
            const uint32_t dst = ring + stage * 2 * CHUNK;
#pragma unroll
            for (int i = 0; i < CHUNK / 512; ++i) {
                const int e = i * 32 + lane, r = e / (D / 8), col = e % (D / 8);
                const int key = chunk * KEYS + r;
                const bool in = key < c.nk;
                const int64_t at = in ? key : 0;
                cp_async_16(dst + piece<D>(r, col), kbase + at * p.ldk + col * 8, in);
                cp_async_16(dst + CHUNK + piece<D>(r, col), vbase + at * p.ldv + col * 8, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&]() {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load(first + i * step, i);
    };
    begin();

    // Q as A fragments: rows lane / 4 and lane / 4 + 8 of the tile
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = tile * kRows + (lane >> 2) + 8 * h;
        const bool in = r < c.nq * p.group;
        const uint16_t* row = p.q + static_cast<int64_t>(c.q0 + (in ? r / p.group : 0)) * p.ldq +
                              (hk * p.group + (in ? r % p.group : 0)) * D + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qa[k][h] = in ? __ldg(reinterpret_cast<const uint32_t*>(row + k * 16)) : 0u;
            qa[k][2 + h] = in ? __ldg(reinterpret_cast<const uint32_t*>(row + k * 16 + 8)) : 0u;
        }
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // a row's maximum (a score) and sum
    // All chunks, with references that are rounded products or exact ones (see kFar).
    // A row of the former whose farthest maximum was too far has to be gone
    // through again: a test in the loop, in front of the exponentials, cost 4 to 15%.
    float farthest = 0.f;
    auto walk = [&](auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
        float ref[2] = {-INFINITY, -INFINITY};  // of m
        int stage = 0;
        for (int chunk = first; chunk < chunks; chunk += step) {
            load(chunk + (STAGES - 1) * step, (stage + STAGES - 1) % STAGES);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t kb = ring + stage * 2 * CHUNK, vb = kb + CHUNK;
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) {  // 32 of D: four 8 x 8 pieces of eight keys
                    uint32_t b[4];
                    ldsm4(b, kb + piece<D>(n * 8 + (lane & 7), k * 4 + (lane >> 3)));
                    mma16816<F16>(sc[n], qa[2 * k], b[0], b[1]);
                    mma16816<F16>(sc[n], qa[2 * k + 1], b[2], b[3]);
                }
            }
            if ((chunk + 1) * KEYS > c.nk) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (chunk * KEYS + n * 8 + (lane & 3) * 2 + (e & 1) >= c.nk) sc[n][e] = -INFINITY;
            }
            // The maximum in use stays until a chunk's is more than 8 above it in the
            // exponent (P is then at most 2^8, fp16 2^15; the final division cancels it).
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mx[0] = fmaxf(mx[0], fmaxf(sc[n][0], sc[n][1]));
                mx[1] = fmaxf(mx[1], fmaxf(sc[n][2], sc[n][3]));
            }
            float alpha[2], off[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                if constexpr (EXACT) {
                    const float up = (mx[h] - m[h]) * p.scale_log2;
                    alpha[h] = up > 8.0f ? ex2(-up) : 1.0f;
                    m[h] = up > 8.0f ? mx[h] : m[h];
                    off[h] = kLift<F16>;
                    if (m[h] > -INFINITY) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            sc[n][2 * h] -= m[h];
                            sc[n][2 * h + 1] -= m[h];
                        }
                    }
                } else {
                    const float mxr = reference<F16>(mx[h], p.scale_log2);
                    const bool up = mxr > ref[h] + 8.0f;
                    off[h] = up ? -mxr : -ref[h];
                    alpha[h] = ex2(ref[h] + off[h]);
                    m[h] = up ? mx[h] : m[h];
                    ref[h] = -off[h];
                    farthest = fmaxf(farthest, fabsf(mxr));
                }
            }
            float add[2] = {0.f, 0.f};
            uint32_t pa[NT / 2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] = ex2(fmaf(sc[n][e], p.scale_log2, off[e >> 1]));
                add[0] += sc[n][0] + sc[n][1];
                add[1] += sc[n][2] + sc[n][3];
                // P is rounded to the 16 bits of V for the product: an element by at
                // most half a step, as V's own values were
                pa[n / 2][(n & 1) * 2] = pack2<F16>(sc[n][0], sc[n][1]);
                pa[n / 2][(n & 1) * 2 + 1] = pack2<F16>(sc[n][2], sc[n][3]);
            }
            l[0] = l[0] * alpha[0] + add[0];
            l[1] = l[1] * alpha[1] + add[1];
            if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[i][0] *= alpha[0];
                    o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1];
                    o[i][3] *= alpha[1];
                }
            }
#pragma unroll
            for (int k = 0; k < NT / 2; ++k) {  // 16 keys
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {  // 16 of D: keys 0-7 and 8-15 of two eights
                    uint32_t b[4];
                    ldsm4_t(b, vb + piece<D>(k * 16 + (lane & 15), i * 2 + (lane >> 4)));
                    mma16816<F16>(o[2 * i], pa[k], b[0], b[1]);
                    mma16816<F16>(o[2 * i + 1], pa[k], b[2], b[3]);
                }
            }
            __syncwarp();
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
    };
    walk(std::false_type{});
    if (__any_sync(0xffffffffu, farthest > kFar)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
        begin();
        walk(std::true_type{});
    }

    // this warp's part: outputs [kRows][D] in its ring, maximum and sum beside them
    float* mine = reinterpret_cast<float*>(smem + warp * S::RING);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = (lane >> 2) + 8 * h;
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) {
            sM[warp * kRows + r] = m[h];
            sL[warp * kRows + r] = l[h];
        }
        if (r < rows) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(mine + r * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        }
    }
    __syncthreads();
    // The warps' parts joined: each row's weights by its maxima, its sum
    // and maximum, then its outputs in the first warp's place.
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        float top = sM[r], sum = 0.f;
#pragma unroll
        for (int i = 1; i < kWarps; ++i) top = fmaxf(top, sM[i * kRows + r]);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float w = sM[i * kRows + r] == -INFINITY ? 0.f : ex2(reference_step<F16>(sM[i * kRows + r], top, p.scale_log2));
            sW[i * kRows + r] = w;
            sum += w * sL[i * kRows + r];
        }
        sTop[r] = top;
        sSum[r] = sum;
    }
    __syncthreads();
    float* joined = reinterpret_cast<float*>(smem);
    const float* parts[kWarps];
#pragma unroll
    for (int i = 0; i < kWarps; ++i) parts[i] = reinterpret_cast<const float*>(smem + i * S::RING);
    for (int e = threadIdx.x; e < rows * (D / 4); e += 32 * kWarps) {
        const int r = e / (D / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float w = sW[i * kRows + r];
            const float4 f = reinterpret_cast<const float4*>(parts[i])[e];
            if (w != 0.f) {
                v.x = fmaf(w, f.x, v.x);
                v.y = fmaf(w, f.y, v.y);
                v.z = fmaf(w, f.z, v.z);
                v.w = fmaf(w, f.w, v.w);
            }
        }
        reinterpret_cast<float4*>(joined)[e] = v;
    }
    // The same over the CTAs of the cluster, in rank order; the loads of all
    // ranks are in flight at once.  Each CTA writes its share of the outputs.
    if (split > 1) cluster_sync();
    else __syncthreads();
    for (int e = rank * 32 * kWarps + threadIdx.x; e < rows * (D / 2); e += split * 32 * kWarps) {
        const int r = e / (D / 2), d = (e % (D / 2)) * 2;
        float a, b, sum, top;
        if (split == 1) {
            a = joined[2 * e];
            b = joined[2 * e + 1];
            sum = sSum[r];
            top = sTop[r];
        } else {
            float w[8], s[8], x[8], y[8];
            top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t to = k < split ? k : 0;
                w[k] = ld_shared_cluster(mapa_shared(smem_u32(sTop + r), to));
                s[k] = ld_shared_cluster(mapa_shared(smem_u32(sSum + r), to));
                x[k] = ld_shared_cluster(mapa_shared(smem_u32(joined + 2 * e), to));
                y[k] = ld_shared_cluster(mapa_shared(smem_u32(joined + 2 * e + 1), to));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < split) top = fmaxf(top, w[k]);
            a = b = sum = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k >= split || w[k] == -INFINITY) {
                    if (k < split) sum += 0.f * s[k];  // NaN stays
                    continue;
                }
                const float f = ex2(reference_step<F16>(w[k], top, p.scale_log2));
                sum = fmaf(f, s[k], sum);
                a = fmaf(f, x[k], a);
                b = fmaf(f, y[k], b);
            }
        }
        const float inv = row_weight(top, sum, c.nk > 0);
        const int row = tile * kRows + r;
        uint16_t* out = p.out + static_cast<int64_t>(c.q0 + row / p.group) * p.ldo + (hk * p.group + row % p.group) * D + d;
        *reinterpret_cast<uint32_t*>(out) = pack2<F16>(a * inv, b * inv);
    }
    if (split > 1) cluster_sync();  // a CTA's part is read until here
}

template <int D, bool F16>
CrossPlan plan_rows(const CrossParams& p, int num_sms) {
    using S = RowsShape<D>;
    static ClusterCounts known = {};
    const int64_t tiles = (static_cast<int64_t>(p.max_q) * p.group + kRows - 1) / kRows;
    const int chunks = (p.max_kv + S::KEYS - 1) / S::KEYS;
    CrossPlan plan = {p.nseq * p.kv_heads * tiles, 1, cudaSuccess};
    // the keys are split over up to eight CTAs while these find room on the SMs
    // and each warp keeps a few chunks
    const int64_t room = static_cast<int64_t>(num_sms) * (D == 256 ? 1 : 2);
    int fit = 0;
    plan.error = clusters_at_once(cross_rows_kernel<D, F16>, 32 * kWarps, S::SMEM, 1, known, fit);
    for (int split = 2; split <= 8 && plan.error == cudaSuccess; split *= 2) {
        if (split * plan.ctas > room || split * kWarps * 2 > chunks) break;
        plan.error = clusters_at_once(cross_rows_kernel<D, F16>, 32 * kWarps, S::SMEM, split, known, fit);
        if (plan.error != cudaSuccess || plan.ctas > fit) break;
        plan.split = split;
    }
    return plan;
}

template <int D, bool F16>
cudaError_t launch_rows(const CrossParams& p, int split, cudaStream_t st) {
    using S = RowsShape<D>;
    auto kern = cross_rows_kernel<D, F16>;
    const int tiles = (p.max_q * p.group + kRows - 1) / kRows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.nseq * split, p.kv_heads * tiles);
    cfg.blockDim = dim3(32 * kWarps);
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
    return cudaLaunchKernelEx(&cfg, kern, p, split);
}

}  // namespace

CrossPlan plan_cross_rows(const CrossParams& p, int head_dim, int num_sms) {
#define RG_CROSS_ROWS(DD)                                         \
    if (head_dim == DD)                                           \
        return p.f16 ? plan_rows<DD, true>(p, num_sms) : plan_rows<DD, false>(p, num_sms);
    RG_CROSS_ROWS(32)
    RG_CROSS_ROWS(64)
    RG_CROSS_ROWS(128)
    RG_CROSS_ROWS(256)
#undef RG_CROSS_ROWS
    return {0, 1, cudaErrorInvalidValue};
}

cudaError_t launch_cross_rows(const CrossParams& p, int head_dim, int split, cudaStream_t st) {
#define RG_CROSS_ROWS(DD)                                         \
    if (head_dim == DD)                                           \
        return p.f16 ? launch_rows<DD, true>(p, split, st) : launch_rows<DD, false>(p, split, st);
    RG_CROSS_ROWS(32)
    RG_CROSS_ROWS(64)
    RG_CROSS_ROWS(128)
    RG_CROSS_ROWS(256)
#undef RG_CROSS_ROWS
    return cudaErrorInvalidValue;
}

}  // namespace rg
