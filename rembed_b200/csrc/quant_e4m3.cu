// quant_e4m3.cu - quantisers of the block-scaled 8-bit floating-point path.
//
// A block is 128 values of one row (activations) or a tile of 128 x 128
// (weights).  With a = max |x| over the block,
//     scale = a / 448   (1 for a block of zeros, never below 2^-126)
//     q = the e4m3 value next to 448 x / a, ties to even
// (next to x / 2^-126 where the scale is that).  The quotient is rounded once,
// from its exact value: a product with a rounded reciprocal would put values
// on the wrong side of a tie, and with 16-bit inputs exact ties are common.
// 16-bit x and a cannot come nearer to a tie than 2^-18 without being one: with
// r + d = 448 / a (r the quotient towards zero, d its remainder's, both once per
// block) and y = x r rounded, y + ((x r - y) + x d) is the quotient to some 2^-30
// of itself or better, and its nearest float says all.  fp32 can come as near as
// 2^-30: the products with r (1 -+ 2^-21) enclose the quotient, and where they
// round to different bytes the value is compared with the midpoint t between the
// two, 448 x with t a, both as exact sums of two floats.
// A NaN in a block makes the scale NaN, an infinity makes it infinite (with
// r = 0: the infinity becomes NaN, the others 0, and 0 * inf is NaN): a
// block that held either is NaN all over once it is scaled back.
//
// Each value is read once into registers, the maximum is found there, and one byte
// is written.  float32 is bound by HBM (98305 x 1024 in 73-82 us, 6.2 TB/s and more;
// 4096 x 4096 in tiles 20 us from a cold cache), 16 bits by the instructions per byte
// (60-66 us, 4.7 TB/s: an instruction issues in 78% of the cycles, DRAM is busy in 52%).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "act16.cuh"
#include "e4m3.cuh"
#include "pdl.cuh"

namespace rg {
namespace {

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// x (r + d) rounded so that its rounding to e4m3 is that of the exact product; the
// remainder is subtracted, so that a zero keeps its sign.
__device__ __forceinline__ float scaled16(float x, float2 inv) {
    const float y = __fmul_rn(x, inv.x);
    return __fsub_rn(y, __fmaf_rn(-x, inv.y, __fmaf_rn(-x, inv.x, y)));
}

// The e4m3 byte of x over a block of maximum a (448 2^-126 at least), given the
// bytes of two values that enclose the quotient: neighbours at most, as the
// enclosure is far narrower than their distance.
__device__ __forceinline__ uint32_t nearer_e4m3(float x, float a, uint32_t lo, uint32_t hi) {
    if (lo == hi) return lo;
    const uint32_t exponent = (lo >> 3) & 15, digits = exponent ? 8 + (lo & 7) : lo & 7;
    // t = (2 digits + 1) 2^(max(exponent, 1) - 11)
    const float t = static_cast<float>(2 * digits + 1) * __uint_as_float((max(exponent, 1u) + 116) << 23);
    // by a power of two, so that neither the products nor their last bits leave the range of floats
    const float by = a >= 1.f ? 0x1p-16f : 0x1p64f;
    const float sx = fabsf(x) * by, sa = a * by;
    // 448 x - t a: the leading parts are near each other, and all four are multiples of 2^-5 of their last bit
    const float px = __fmul_rn(kE4Max, sx), pa = __fmul_rn(t, sa);
    const float diff = __fadd_rn(__fadd_rn(px, -pa), __fadd_rn(__fmaf_rn(kE4Max, sx, -px), -__fmaf_rn(t, sa, -pa)));
    return diff > 0.f || (diff == 0.f && (lo & 1)) ? hi : lo;
}

// Two values as e4m3, to nearest, ties to even, clamped to +-448; the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

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
    // Rows aligned to nothing but the element, and the matrix's edges: values l,
    // l + LANES, ... of the first n of a block (zeros behind them), so that a load
    // of the lanes is contiguous.
    static __device__ __forceinline__ uint4 load_strided(const void* block, int l, int n) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (l + i * LANES >= n) continue;
            if constexpr (E == Elem::kF32)
                w[i] = __ldg(static_cast<const uint32_t*>(block) + l + i * LANES);
            else
                w[i >> 1] |= static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(block) + l + i * LANES)) << (16 * (i & 1));
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // The larger of two pairs of 16-bit values, NaN if one is.
    static __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
        uint32_t y;
        if constexpr (E == Elem::kF16)
            asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
        else
            asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
        return y;
    }
    // max |x| of the V values, NaN if one is (as bits, which order like the values)
    static __device__ __forceinline__ uint32_t max_bits(const uint4& u) {
        if constexpr (E == Elem::kF32) {
            float f[V];
            unpack(u, f);
            float m = fabsf(f[0]);
#pragma unroll
            for (int i = 1; i < V; ++i) m = max_nan(m, fabsf(f[i]));
            return __float_as_uint(m);
        } else {
            const uint32_t mask = 0x7fff7fffu;
            const float2 p = unpack2<E == Elem::kF16>(
                max_pair(max_pair(u.x & mask, u.y & mask), max_pair(u.z & mask, u.w & mask)));
            return __float_as_uint(max_nan(p.x, p.y));
        }
    }
    // The V values over their scale as e4m3 bytes.
    static __device__ __forceinline__ void convert(const uint4& u, float2 inv, uint32_t (&w)[V / 4]) {
        float f[V];
        unpack(u, f);
        if constexpr (E == Elem::kF32) {
            // between these two products lies the exact one; a midpoint between them is rare
            const float lo = inv.x * (1.0f - 0x1p-21f), hi = inv.x * (1.0f + 0x1p-21f);
            w[0] = to_e4m3x2(f[0] * lo, f[1] * lo) | to_e4m3x2(f[2] * lo, f[3] * lo) << 16;
            const uint32_t v = to_e4m3x2(f[0] * hi, f[1] * hi) | to_e4m3x2(f[2] * hi, f[3] * hi) << 16;
            if (w[0] == v) return;
            uint32_t q = 0u;
#pragma unroll
            for (int i = 0; i < V; ++i) q |= nearer_e4m3(f[i], inv.y, (w[0] >> (8 * i)) & 255, (v >> (8 * i)) & 255) << (8 * i);
            w[0] = q;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = scaled16(f[i], inv);
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                w[i] = to_e4m3x2(f[4 * i], f[4 * i + 1]) | to_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16;
        }
    }
    // A whole block's values as the two loads took them: from column l of it.
    static __device__ __forceinline__ void store_whole(uint8_t* block, int l, const uint4& u, float2 inv) {
        uint32_t w[V / 4];
        convert(u, inv, w);
        if constexpr (V == 8)
            *reinterpret_cast<uint2*>(block + l) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(block + l) = w[0];
    }
    static __device__ __forceinline__ void store_strided(uint8_t* block, int l, int n, const uint4& u, float2 inv) {
        uint32_t w[V / 4];
        convert(u, inv, w);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (l + i * LANES < n) block[l + i * LANES] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
    }
};

// A block's scale from the bits of its maximum a, and what the conversion needs of
// its reciprocal: r, and d (16 bits) or a (fp32, at least 448 2^-126).
template <Elem E>
__device__ __forceinline__ float block_scale(uint32_t max_bits, float2& inv) {
    const float a = __uint_as_float(max_bits);
    constexpr float kLeast = 0x1p-126f;
    if (a == 0.f) {
        inv = make_float2(1.f, E == Elem::kF32 ? kE4Max : 0.f);
        return 1.f;
    }
    const float s = a / kE4Max;
    if (s < kLeast) {
        inv = make_float2(0x1p126f, E == Elem::kF32 ? kE4Max * kLeast : 0.f);
        return kLeast;
    }
    const float r = __fdiv_rz(kE4Max, a);
    if constexpr (E == Elem::kF32)
        inv = make_float2(r, a);
    else
        inv = make_float2(r, isinf(a) ? 0.f : __fmaf_rn(-r, a, kE4Max) / a);  // a NaN stays
    return s;
}

// A warp takes one block column of eight rows (float32: eight warp-wide loads,
// 16-bit: four).  All loads are in flight before the first maximum, and the
// rows' scales, neighbours in memory, leave as one 32-byte sector.
template <Elem E>
constexpr int kGroup = 8 / Lane<E>::ROWS;
constexpr int kRowWarps = 8;

// How a warp's rows lie: at the edge of the matrix, or whole blocks in rows that
// are 16-byte aligned or not.
enum class Part { kEdge, kAligned, kUnaligned };

template <Elem E, Part P>
__device__ __forceinline__ void quantize_rows_group(const QuantE4Params& p, int64_t first, int b, int lane) {
    using L = Lane<E>;
    const int rows = P != Part::kEdge ? 8
                          : static_cast<int>(min(static_cast<int64_t>(8), p.rows - first));
    // a row may be wider than 2^31 bytes
    const int64_t col0 = static_cast<int64_t>(b) * kE4Block, c = col0 + (lane % L::LANES) * L::V;
    const int behind = static_cast<int>(min(static_cast<int64_t>(kE4Block), p.K - col0));  // columns from col0 on
    const int mine = lane / L::LANES;  // row of the warp-wide load
    const uint8_t* src = static_cast<const uint8_t*>(p.x) + (first + mine) * p.ldx * L::BYTES;
    uint8_t* dst = p.q + (first + mine) * p.ldq;
    const int64_t src_step = L::ROWS * p.ldx * L::BYTES, dst_step = L::ROWS * p.ldq;
    uint4 u[kGroup<E>];
#pragma unroll
    for (int i = 0; i < kGroup<E>; ++i) {
        if constexpr (P == Part::kAligned) {
            u[i] = __ldg(reinterpret_cast<const uint4*>(src + i * src_step + c * L::BYTES));
        } else if constexpr (P == Part::kUnaligned) {
            u[i] = L::load_strided(src + i * src_step + col0 * L::BYTES, lane % L::LANES, kE4Block);
        } else {
            u[i] = make_uint4(0u, 0u, 0u, 0u);
            if (i * L::ROWS + mine < rows)
                u[i] = L::load_strided(src + i * src_step + col0 * L::BYTES, lane % L::LANES, behind);
        }
    }
    // lane `row of the group` takes that row's maximum through the divisions
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kGroup<E>; ++i) {
        uint32_t m = L::max_bits(u[i]);
        if constexpr (L::ROWS == 1) {
            m = __reduce_max_sync(0xffffffffu, m);
            top = lane == i ? m : top;
        } else {
#pragma unroll
            for (int o = L::LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const uint32_t other = __shfl_xor_sync(0xffffffffu, m, L::LANES);
            if (lane / 2 == i) top = (lane & 1) == mine ? m : other;
        }
    }
    float2 inv;
    const float s = block_scale<E>(top, inv);
    if (lane < rows) p.scale[b * p.ld_scale + first + lane] = s;
#pragma unroll
    for (int i = 0; i < kGroup<E>; ++i) {
        const float2 f = make_float2(__shfl_sync(0xffffffffu, inv.x, i * L::ROWS + mine),
                                     __shfl_sync(0xffffffffu, inv.y, i * L::ROWS + mine));
        if constexpr (P == Part::kAligned) {
            L::store_whole(dst + i * dst_step, c, u[i], f);
        } else if constexpr (P == Part::kUnaligned) {
            L::store_strided(dst + i * dst_step + col0, lane % L::LANES, kE4Block, u[i], f);
        } else {
            if (i * L::ROWS + mine < rows)
                L::store_strided(dst + i * dst_step + col0, lane % L::LANES, behind, u[i], f);
        }
    }
}

template <Elem E>
__global__ void __launch_bounds__(32 * kRowWarps) quantize_rows_e4m3_kernel(QuantE4Params p, bool aligned) {
    constexpr int kRowsOf = 8;
    pdl_trigger();
    pdl_wait();
    const int kb = (p.K + kE4Block - 1) / kE4Block;
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
    const int64_t group = item / kb;
    const int b = static_cast<int>(item - group * kb);
    const int64_t first = group * kRowsOf;
    if (first >= p.rows) return;
    if (first + kRowsOf > p.rows || (b + 1) * kE4Block > p.K)
        quantize_rows_group<E, Part::kEdge>(p, first, b, lane);
    else if (aligned)
        quantize_rows_group<E, Part::kAligned>(p, first, b, lane);
    else
        quantize_rows_group<E, Part::kUnaligned>(p, first, b, lane);
}

// One CTA per 128 x 128 tile, held in registers.
constexpr int kTileWarps = 16;

template <Elem E, Part P>
__device__ __forceinline__ void quantize_tile(const QuantE4Params& p, int64_t first, int64_t col0) {
    using L = Lane<E>;
    constexpr int LOADS = kE4Block / (kTileWarps * L::ROWS);
    __shared__ uint32_t part[kTileWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = col0 + (lane % L::LANES) * L::V;  // a row may be wider than 2^31 bytes
    const int behind = static_cast<int>(min(static_cast<int64_t>(kE4Block), p.K - col0));  // columns from col0 on
    const int64_t r0 = first + warp * L::ROWS + lane / L::LANES;
    const uint8_t* src = static_cast<const uint8_t*>(p.x) + r0 * p.ldx * L::BYTES;
    uint8_t* dst = p.q + r0 * p.ldq;
    const int64_t src_step = kTileWarps * L::ROWS * p.ldx * L::BYTES, dst_step = kTileWarps * L::ROWS * p.ldq;
    uint4 u[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        if constexpr (P == Part::kAligned) {
            u[i] = __ldg(reinterpret_cast<const uint4*>(src + i * src_step + c * L::BYTES));
        } else if constexpr (P == Part::kUnaligned) {
            u[i] = L::load_strided(src + i * src_step + col0 * L::BYTES, lane % L::LANES, kE4Block);
        } else {
            u[i] = make_uint4(0u, 0u, 0u, 0u);
            if (r0 + i * kTileWarps * L::ROWS < p.rows)
                u[i] = L::load_strided(src + i * src_step + col0 * L::BYTES, lane % L::LANES, behind);
        }
    }
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) m = max(m, L::max_bits(u[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) part[warp] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, part[lane & (kTileWarps - 1)]);
    float2 inv;
    const float s = block_scale<E>(m, inv);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        if constexpr (P == Part::kAligned) {
            L::store_whole(dst + i * dst_step, c, u[i], inv);
        } else if constexpr (P == Part::kUnaligned) {
            L::store_strided(dst + i * dst_step + col0, lane % L::LANES, kE4Block, u[i], inv);
        } else {
            if (r0 + i * kTileWarps * L::ROWS < p.rows)
                L::store_strided(dst + i * dst_step + col0, lane % L::LANES, behind, u[i], inv);
        }
    }
    if (threadIdx.x == 0) p.scale[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <Elem E>
__global__ void __launch_bounds__(32 * kTileWarps) quantize_tiles_e4m3_kernel(QuantE4Params p, bool aligned) {
    pdl_trigger();
    pdl_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.y) * kE4Block;
    const int64_t col0 = static_cast<int64_t>(blockIdx.x) * kE4Block;
    if (first + kE4Block > p.rows || col0 + kE4Block > p.K)
        quantize_tile<E, Part::kEdge>(p, first, col0);
    else if (aligned)
        quantize_tile<E, Part::kAligned>(p, first, col0);
    else
        quantize_tile<E, Part::kUnaligned>(p, first, col0);
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
    const int64_t warps = (static_cast<int64_t>(p.rows) + 7) / 8 * kb;
    const int64_t grid = (warps + kRowWarps - 1) / kRowWarps;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_pdl(quantize_rows_e4m3_kernel<E>, dim3(static_cast<unsigned>(grid)), dim3(32 * kRowWarps), 0, st, p,
                      aligned_x<E>(p) && aligned_q<E>(p));
}

template <Elem E>
cudaError_t tiles_of(const QuantE4Params& p, cudaStream_t st) {
    const dim3 grid((p.K + kE4Block - 1) / kE4Block, (p.rows + kE4Block - 1) / kE4Block);
    if (grid.y > 65535) return cudaErrorInvalidValue;
    return launch_pdl(quantize_tiles_e4m3_kernel<E>, grid, dim3(32 * kTileWarps), 0, st, p, aligned_x<E>(p) && aligned_q<E>(p));
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
