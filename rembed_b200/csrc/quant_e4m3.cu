// quant_e4m3.cu - quantisers of the block-scaled 8-bit floating-point path.
//
// A block is 128 values of one row (activations) or a tile of 128 x 128
// (weights).  With a = max |x| over the block,
//     s = a / 448      (1 for a block of zeros, never below 2^-126)
//     q = e4m3(x * (1 / s)), to nearest, ties to even, clamped to +-448
// so that q * s is within half an e4m3 step of x.  The maximum is taken on the
// bit patterns of |x| as unsigned integers, where a NaN orders above infinity:
// a block with a NaN gets the scale NaN, one with an infinity the scale
// infinity (then x * 0 is NaN for the infinity and 0 elsewhere, and 0 * inf
// is NaN), so a block that held either is NaN all over once it is scaled back.
//
// Both kernels are bound by HBM: each value is read once into registers, the
// maximum is found there, and one byte is written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "act16.cuh"
#include "e4m3.cuh"
#include "pdl.cuh"

namespace rg {
namespace {

// One lane's 16 bytes of a block's row: V values, LANES lanes a row.
template <Elem E>
struct Lane {
    static constexpr int BYTES = E == Elem::kF32 ? 4 : 2;
    static constexpr int V = 16 / BYTES;
    static constexpr int LANES = kE4Block / V;
    static constexpr int ROWS = 32 / LANES;  // rows one warp-wide load covers

    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[V]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (E == Elem::kF32) {
                f[i] = __uint_as_float(w[i]);
            } else {
                const float2 p = unpack2<E == Elem::kF16>(w[i]);
                f[2 * i] = p.x;
                f[2 * i + 1] = p.y;
            }
        }
    }
    // The V values from column c of a row (`row` its first value); columns
    // from K on read as zeros.  vec: 16-byte aligned rows.
    static __device__ __forceinline__ uint4 load(const void* row, int c, int K, bool vec) {
        if (vec && c + V <= K)
            return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + static_cast<int64_t>(c) * BYTES));
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (c + i >= K) break;
            if constexpr (E == Elem::kF32)
                w[i] = __ldg(static_cast<const uint32_t*>(row) + c + i);
            else
                w[i >> 1] |= static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(row) + c + i)) << (16 * (i & 1));
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ uint32_t max_bits(const uint4& u) {
        float f[V];
        unpack(u, f);
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
        return m;
    }
    // The V values times inv as e4m3 bytes to columns c.. of a row.
    static __device__ __forceinline__ void store(uint8_t* row, int c, int K, bool vec, const uint4& u, float inv) {
        if (c >= K) return;
        float f[V];
        unpack(u, f);
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const uint32_t lo =
                __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] * inv, f[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi =
                __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] * inv, f[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            w[i] = lo | (hi << 16);
        }
        if (vec && c + V <= K) {
            if constexpr (V == 8)
                *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t*>(row + c) = w[0];
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < K) row[c + i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
    }
};

__device__ __forceinline__ float block_scale(uint32_t max_bits) {
    if (max_bits == 0u) return 1.0f;
    const float s = __uint_as_float(max_bits) / kE4Max;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;  // a NaN stays
}

// A warp takes one block column of kGroup warp-wide loads of rows: 8 rows of
// float32, 16 of a 16-bit type.  All loads are in flight before the first
// maximum, and the rows' scales, neighbours in memory, leave in one store of
// at least a 32-byte sector.
constexpr int kGroup = 8;
constexpr int kRowWarps = 8;

template <Elem E>
__global__ void __launch_bounds__(32 * kRowWarps) quantize_rows_e4m3_kernel(QuantE4Params p, bool vec_x, bool vec_q) {
    using L = Lane<E>;
    pdl_trigger();
    pdl_wait();
    const int kb = (p.K + kE4Block - 1) / kE4Block;
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
    const int64_t group = item / kb;
    const int b = static_cast<int>(item - group * kb);
    const int64_t r0 = group * (kGroup * L::ROWS) + lane / L::LANES;
    if (r0 - lane / L::LANES >= p.rows) return;
    const int c = b * kE4Block + (lane % L::LANES) * L::V;
    uint4 u[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        const int64_t r = r0 + i * L::ROWS;
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < p.rows) u[i] = L::load(static_cast<const uint8_t*>(p.x) + r * p.ldx * L::BYTES, c, p.K, vec_x);
    }
    float mine = 1.0f;  // the scale this lane stores: row `lane` of the group
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        uint32_t m = L::max_bits(u[i]);
#pragma unroll
        for (int o = L::LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = block_scale(m);
        const int64_t r = r0 + i * L::ROWS;
        if (r < p.rows) L::store(p.q + r * p.ldq, c, p.K, vec_q, u[i], 1.0f / s);
#pragma unroll
        for (int j = 0; j < L::ROWS; ++j) {
            const float sj = __shfl_sync(0xffffffffu, s, j * L::LANES);
            if (lane == i * L::ROWS + j) mine = sj;
        }
    }
    const int64_t r = group * (kGroup * L::ROWS) + lane;
    if (lane < kGroup * L::ROWS && r < p.rows) p.scale[b * p.ld_scale + r] = mine;
}

// One CTA per 128 x 128 tile, held in registers (64 bytes of a row's block a
// warp-wide load, 16 or 8 loads a thread).
template <Elem E>
__global__ void __launch_bounds__(256) quantize_tiles_e4m3_kernel(QuantE4Params p, bool vec_x, bool vec_q) {
    using L = Lane<E>;
    constexpr int LOADS = kE4Block / (8 * L::ROWS);
    __shared__ uint32_t part[8];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * kE4Block + (lane % L::LANES) * L::V;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kE4Block + warp * L::ROWS + lane / L::LANES;
    uint4 u[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int64_t r = r0 + i * 8 * L::ROWS;
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < p.rows) u[i] = L::load(static_cast<const uint8_t*>(p.x) + r * p.ldx * L::BYTES, c, p.K, vec_x);
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) m = max(m, L::max_bits(u[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) part[warp] = m;
    __syncthreads();
    m = part[lane & 7];
    m = __reduce_max_sync(0xffffffffu, m);
    const float s = block_scale(m);
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int64_t r = r0 + i * 8 * L::ROWS;
        if (r < p.rows) L::store(p.q + r * p.ldq, c, p.K, vec_q, u[i], inv);
    }
    if (threadIdx.x == 0) p.scale[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <Elem E>
bool aligned_x(const QuantE4Params& p) {
    return reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx % Lane<E>::V == 0;
}
template <Elem E>
bool aligned_q(const QuantE4Params& p) {
    return reinterpret_cast<uintptr_t>(p.q) % Lane<E>::V == 0 && p.ldq % Lane<E>::V == 0;
}

template <Elem E>
cudaError_t rows_of(const QuantE4Params& p, cudaStream_t st) {
    const int64_t kb = (p.K + kE4Block - 1) / kE4Block;
    const int64_t rows = kGroup * Lane<E>::ROWS;
    const int64_t warps = (p.rows + rows - 1) / rows * kb;
    const int64_t grid = (warps + kRowWarps - 1) / kRowWarps;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_pdl(quantize_rows_e4m3_kernel<E>, dim3(static_cast<unsigned>(grid)), dim3(32 * kRowWarps), 0, st, p,
                      aligned_x<E>(p), aligned_q<E>(p));
}

template <Elem E>
cudaError_t tiles_of(const QuantE4Params& p, cudaStream_t st) {
    const dim3 grid((p.K + kE4Block - 1) / kE4Block, (p.rows + kE4Block - 1) / kE4Block);
    if (grid.y > 65535) return cudaErrorInvalidValue;
    return launch_pdl(quantize_tiles_e4m3_kernel<E>, grid, dim3(256), 0, st, p, aligned_x<E>(p), aligned_q<E>(p));
}

}  // namespace

cudaError_t launch_quantize_rows_e4m3(Elem type, const QuantE4Params& p, cudaStream_t st) {
    switch (type) {
    case Elem::kF32: return rows_of<Elem::kF32>(p, st);
    case Elem::kF16: return rows_of<Elem::kF16>(p, st);
    case Elem::kBF16: return rows_of<Elem::kBF16>(p, st);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_quantize_tiles_e4m3(Elem type, const QuantE4Params& p, cudaStream_t st) {
    switch (type) {
    case Elem::kF32: return tiles_of<Elem::kF32>(p, st);
    case Elem::kF16: return tiles_of<Elem::kF16>(p, st);
    case Elem::kBF16: return tiles_of<Elem::kBF16>(p, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace rg
