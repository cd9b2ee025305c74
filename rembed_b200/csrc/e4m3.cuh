// e4m3.cuh - the block-scaled 8-bit floating-point path: quantisers and the
// matrix product over e4m3 operands with a float32 scale per block of 128.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace rg {

constexpr int kE4Block = 128;       // values of K (and weight rows) that share a scale
constexpr float kE4Max = 448.0f;    // largest finite e4m3 value

// Element type of the unquantised side, as RG_DTYPE_* number it.
enum class Elem : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// x [rows x K], row stride ldx -> q [rows x K] e4m3, row stride ldq.
// rows: scale[b * ld_scale + r] for block b of row r.
// tiles: scale[(r / 128) * ceil(K / 128) + b] for each 128 x 128 tile.
struct QuantE4Params {
    const void* x;
    int64_t ldx;
    int rows, K;
    uint8_t* q;
    int64_t ldq;
    float* scale;
    int64_t ld_scale;
};
cudaError_t launch_quantize_rows_e4m3(Elem type, const QuantE4Params& p, cudaStream_t st);
cudaError_t launch_quantize_tiles_e4m3(Elem type, const QuantE4Params& p, cudaStream_t st);

// y[m][n] = sum_b x_scale[b][m] * w_scale[n / 128][b] * sum_{k in block b}
//           xq[m][k] * wq[n][k]  (+ bias[n]).
struct DenseE4Params {
    const uint8_t *xq, *wq;      // e4m3 [M x K], [N x K]
    int64_t ldx, ldw;            // row strides, multiples of 16
    const float* x_scale;        // [ceil(K / 128) x ld_xs]
    int64_t ld_xs;
    const float* w_scale;        // [ceil(N / 128) x ceil(K / 128)]
    const float* bias;           // [N] or nullptr
    void* y;
    int64_t ldy;
    int M, N, K;
    int* status;
};
cudaError_t launch_dense_e4m3(Elem out, const DenseE4Params& p, int num_sms, cudaStream_t st);

}  // namespace rg
