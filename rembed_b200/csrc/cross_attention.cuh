// cross_attention.cuh - attention of packed query sequences to the keys and
// values of other sequences (an encoder's states), each of its own length.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rg {

// attention_tc.cu: tensor map over a 16-bit matrix of `rows` x `cols` at row
// stride ld, boxes of 64 columns (128 bytes, 128-byte swizzle) x box_rows.
bool make_rows_tmap(CUtensorMap* map, const void* base, bool f16, uint64_t rows, uint64_t cols, uint64_t ld,
                    uint32_t box_rows);

// Query sequence s: rows [cu_q[s], cu_q[s + 1]) of q and out; its keys and
// values: rows [kv_begin[s], kv_begin[s] + kv_len[s]) of k and v.  Query head h
// at columns h * D, key/value head h / group.
struct CrossParams {
    const uint16_t *q, *k, *v;
    bool f16;
    int ldq, ldk, ldv;
    const int32_t *cu_q, *kv_begin, *kv_len;
    int nseq, Tq, Tk, max_q, max_kv;
    int heads, kv_heads, group;
    float scale_log2;  // scale * log2(e), positive
    uint16_t* out;
    int ldo;
    int* status;
};

// One query sequence's part, read on the device; false (with the status bits
// `raise`) if it does not lie within the buffers and the given longest lengths.
struct CrossSeq {
    int q0, nq, k0, nk;
};
#ifdef __CUDACC__
__device__ __forceinline__ bool cross_seq(const CrossParams& p, int s, CrossSeq& c, int raise) {
    c.q0 = __ldg(p.cu_q + s);
    const int q1 = __ldg(p.cu_q + s + 1);
    c.k0 = __ldg(p.kv_begin + s);
    c.nk = __ldg(p.kv_len + s);
    c.nq = q1 - c.q0;
    const bool ok = c.q0 >= 0 && q1 >= c.q0 && q1 <= p.Tq && c.nq <= p.max_q && c.nk >= 0 && c.nk <= p.max_kv &&
                    c.k0 >= 0 && c.k0 <= p.Tk - c.nk;
    if (!ok && raise) atomicOr(p.status, raise);
    return ok;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A key's exponent is its score x times scale less its row's reference, which is the
// same for all of the row's keys and cancels.  While the score m in use for the
// maximum has |m scale| up to 2^10, the reference is that product, rounded.
// Beyond, the rounding would come to reach the size of the exponents, or the
// product is not finite: there it is the exact product, and the exponent (x - m)
// scale.  A row that goes from one to the other mixes exponents 2^-14 apart.
// fp16 has no steps below 2^-24, and a long text many probabilities down there:
// its exponents are 7 higher (probabilities up to 2^15; 8 of that is how far a
// maximum may be above the one in use).
constexpr float kFar = 0x1p10f;
template <bool F16>
constexpr float kLift = F16 ? 7.0f : 0.0f;
template <bool F16>
__device__ __forceinline__ float reference(float m, float scale) {
    return F16 ? __fmaf_rn(m, scale, -kLift<F16>) : __fmul_rn(m, scale);
}
// The maximum of a row's next keys, mx, into m and its reference ref, where the
// larger one's reference is far; weights so far count alpha times from here on.
template <bool F16>
__device__ __forceinline__ void far_maximum(float mx, float scale, float& m, float& ref, float& alpha) {
    const bool near = fabsf(ref) <= kFar;
    const float up = (mx - m) * scale;
    alpha = 1.0f;
    if (near || up > 8.0f) {
        alpha = ex2(near ? ref - reference<F16>(mx, scale) : -up);
        m = mx;
        ref = reference<F16>(mx, scale);
    }
}
// By how much the reference of m = a is above that of m = b.
template <bool F16>
__device__ __forceinline__ float reference_step(float a, float b, float scale) {
    const float ra = reference<F16>(a, scale), rb = reference<F16>(b, scale);
    return fabsf(ra) > kFar && fabsf(rb) > kFar ? (a - b) * scale : ra - rb;
}
// What a row's products are multiplied by at the end, from its maximum and sum: no
// key gives zeros, keys with scores of -infinity alone 0 / 0; a NaN stays.
__device__ __forceinline__ float row_weight(float m, float sum, bool keys) {
    return m > -INFINITY ? 1.0f / sum : __int_as_float(keys ? 0x7fffffff : 0);
}
#endif

// What a kernel would do with a call: CTAs before the keys are split, and over
// how many CTAs of a cluster they are.
struct CrossPlan {
    int64_t ctas;
    int split;
    cudaError_t error;
};

// Few query rows per key/value head (one or a few tokens): bound by reading K and V.
CrossPlan plan_cross_rows(const CrossParams& p, int head_dim, int num_sms);
cudaError_t launch_cross_rows(const CrossParams& p, int head_dim, int split, cudaStream_t st);
// Any number of query rows: tiles of 128 on the tensor cores of tcgen05.
CrossPlan plan_cross_tiles(const CrossParams& p, int head_dim, int num_sms);
cudaError_t launch_cross_tiles(const CrossParams& p, int head_dim, int split, cudaStream_t st);
// The one of the two that suits the call.
cudaError_t launch_cross(const CrossParams& p, int head_dim, int num_sms, cudaStream_t st);

}  // namespace rg
