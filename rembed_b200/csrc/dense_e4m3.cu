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

#include "act16.cuh"
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
// Weight rows on the M side of the MMA: a CTA owns 128 weight rows (one
// weight block, so its weight scale is one number per block of K) and NT rows
// of x.  Roles (256 threads):
//   warp 0     TMA producer: 128 weight rows and NT x rows of each k-block;
//   warp 1     MMA issuer (one thread), four MMAs per k-block into one of ACC
//              accumulators;
//   warp 2     TMEM allocator, then the scales: xs * ws of each k-block into
//              a ring in shared memory;
//   warps 4-7  accumulation, thread = weight row = TMEM lane, NT sums each;
//              the stores of a warp are 32 neighbouring columns of y.
template <int NT>
struct ThinShape {
    static constexpr int A_BYTES = 128 * 128, B_BYTES = NT * 128;
    static constexpr int STAGES = NT == 128 ? 6 : 8;
    static constexpr int ACC = NT == 128 ? 2 : 4;
    static constexpr uint32_t TMEM_COLS = ACC * NT < 32 ? 32 : ACC * NT;
    static constexpr int SR = 8;  // ring of scales
    static constexpr int SMEM = STAGES * (A_BYTES + B_BYTES) + SR * NT * 4 + 1024 + 512;
    static constexpr int THREADS = 256;
};

template <int NT, Elem O>
__global__ void __launch_bounds__(256, 1)
    dense_e4m3_thin_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           DenseE4Params p) {
    using S = ThinShape<NT>;
    constexpr int STAGES = S::STAGES, ACC = S::ACC, SR = S::SR;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * S::A_BYTES;
    float* sScale = reinterpret_cast<float*>(sB + STAGES * S::B_BYTES);  // [SR][NT]
    uint64_t* full = reinterpret_cast<uint64_t*>(sScale + SR * NT);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + ACC;
    uint64_t* cfull = tempty + ACC;
    uint64_t* cempty = cfull + SR;
    uint64_t* drain = cempty + SR;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kblocks = (p.K + kE4Block - 1) / kE4Block;
    const int nb = blockIdx.x, n0 = nb * 128, m0 = blockIdx.y * NT;

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
            mbar_init(&cfull[s], 1);
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

    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            for (int kb = 0; kb < kblocks; ++kb) {
                const int s = kb % STAGES;
                if (!mbar_wait(&empty[s], ((kb / STAGES) & 1) ^ 1, p.status, abort_flag)) break;
                mbar_arrive_expect_tx(&full[s], S::A_BYTES + S::B_BYTES);
                tma_load_2d(sA + s * S::A_BYTES, &tmW, &full[s], kb * 128, n0);
                tma_load_2d(sB + s * S::B_BYTES, &tmX, &full[s], kb * 128, m0);
                issued = kb + 1;
            }
            // every load issued has landed before the CTA may exit
            for (int kb = issued > STAGES ? issued - STAGES : 0; kb < issued; ++kb)
                mbar_drain(&full[kb % STAGES], (kb / STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_e4m3(128, NT);
            bool issued = false;
            for (int kb = 0; kb < kblocks; ++kb) {
                const int s = kb % STAGES, a = kb % ACC;
                if (!mbar_wait(&tempty[a], ((kb / ACC) & 1) ^ 1, p.status, abort_flag) ||
                    !mbar_wait(&full[s], (kb / STAGES) & 1, p.status, abort_flag))
                    break;
                tc_fence_after();
                const uint64_t ad = sdesc_k128(smem_u32(sA + s * S::A_BYTES));
                const uint64_t bd = sdesc_k128(smem_u32(sB + s * S::B_BYTES));
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + a * NT, ad + 2 * k, bd + 2 * k, idesc, k > 0);
                issued = true;
                umma_commit(&empty[s]);
                umma_commit(&tfull[a]);
            }
            if (issued) {
                umma_commit(drain);
                mbar_drain(drain, 0);
            }
        }
    } else if (warp == 2) {
        const float* ws = p.w_scale + static_cast<int64_t>(nb) * kblocks;
        for (int kb = 0; kb < kblocks; ++kb) {
            const int c = kb % SR;
            const float w = __ldg(ws + kb);
            float v[(NT + 31) / 32];
#pragma unroll
            for (int i = 0; i < (NT + 31) / 32; ++i) {
                const int m = m0 + lane + 32 * i;
                v[i] = m < p.M && lane + 32 * i < NT ? __ldg(p.x_scale + kb * p.ld_xs + m) * w : 0.f;
            }
            if (!mbar_wait(&cempty[c], ((kb / SR) & 1) ^ 1, p.status, abort_flag)) break;
#pragma unroll
            for (int i = 0; i < (NT + 31) / 32; ++i)
                if (lane + 32 * i < NT) sScale[c * NT + lane + 32 * i] = v[i];
            __syncwarp();
            if (lane == 0) mbar_arrive(&cfull[c]);
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3;
        const int n = n0 + quarter * 32 + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        float acc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = 0.f;
        bool ok = true;
        for (int kb = 0; kb < kblocks; ++kb) {
            const int a = kb % ACC, c = kb % SR;
            if (!mbar_wait(&cfull[c], (kb / SR) & 1, p.status, abort_flag) ||
                !mbar_wait(&tfull[a], (kb / ACC) & 1, p.status, abort_flag)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const float4* sc = reinterpret_cast<const float4*>(sScale + c * NT);
#pragma unroll
            for (int h = 0; h < NT / 16; ++h) {
                uint32_t t[16];
                tmem_ld16(tmem + lane_addr + a * NT + h * 16, t);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 s4 = sc[h * 4 + i];
                    acc[h * 16 + 4 * i + 0] = fmaf(__uint_as_float(t[4 * i + 0]), s4.x, acc[h * 16 + 4 * i + 0]);
                    acc[h * 16 + 4 * i + 1] = fmaf(__uint_as_float(t[4 * i + 1]), s4.y, acc[h * 16 + 4 * i + 1]);
                    acc[h * 16 + 4 * i + 2] = fmaf(__uint_as_float(t[4 * i + 2]), s4.z, acc[h * 16 + 4 * i + 2]);
                    acc[h * 16 + 4 * i + 3] = fmaf(__uint_as_float(t[4 * i + 3]), s4.w, acc[h * 16 + 4 * i + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&tempty[a]);
                mbar_arrive(&cempty[c]);
            }
        }
        if (ok && n < p.N) {
            const float b = p.bias ? __ldg(p.bias + n) : 0.f;
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int m = m0 + i;
                const float v = acc[i] + b;
                if (m < p.M) {
                    store_y<O>(p.y, m * p.ldy + n, v);
                    amax = fmaxf(amax, fabsf(v));
                }
            }
            if (O == Elem::kF16 && amax > 65504.0f) atomicOr(p.status, kStatusF16Overflow);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, S::TMEM_COLS);
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

template <int NT, Elem O>
cudaError_t launch_thin(const DenseE4Params& p, cudaStream_t st) {
    using S = ThinShape<NT>;
    static unsigned configured = 0;
    auto kern = dense_e4m3_thin_kernel<NT, O>;
    cudaError_t e = allow_smem(kern, S::SMEM, configured);
    if (e != cudaSuccess) return e;
    CUtensorMap tw, tx;
    if (!make_kmajor_tmap(&tw, p.wq, 1, p.N, p.K, p.ldw, 128) || !make_kmajor_tmap(&tx, p.xq, 1, p.M, p.K, p.ldx, NT))
        return cudaErrorInvalidValue;
    const dim3 grid((p.N + 127) / 128, (p.M + NT - 1) / NT);
    return launch_pdl(kern, grid, dim3(S::THREADS), S::SMEM, st, tw, tx, p);
}

template <Elem O>
cudaError_t launch_out(const DenseE4Params& p, int num_sms, cudaStream_t st) {
    if (p.M <= 16) return launch_thin<16, O>(p, st);
    if (p.M <= 32) return launch_thin<32, O>(p, st);
    if (p.M <= 64) return launch_thin<64, O>(p, st);
    return launch_thin<128, O>(p, st);
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
