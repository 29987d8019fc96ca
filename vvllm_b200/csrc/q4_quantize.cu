// q4_quantize.cu -- 4-bit group quantization of weights (fp32 or bf16) and its inverse.
//
// Per group of `group` consecutive weights of a row: s = bf16(max |w| / 7) with NaN skipped,
// q = round(w / s) (ties to even) within -8..7 (q4_common.cuh).  Deterministic and exact, so the
// codes of a matrix are a function of its values alone.
//
// Dequantization writes q * s for all rows, or for a list of rows: the token lookup of a tied
// embedding / output head that is kept in 4 bits.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "q4_common.cuh"

namespace b200q8 {

namespace {

__device__ __forceinline__ float src_f32(const float* p) { return *p; }
__device__ __forceinline__ float src_f32(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// Any K, any alignment: a warp per group, at most four weights a lane.
template <typename WT>
__global__ void __launch_bounds__(256) q4_quantize_generic_kernel(const WT* __restrict__ w, uint8_t* __restrict__ q4,
                                                                  uint16_t* __restrict__ scales, long long groups,
                                                                  int ng, long long K, int group)
{
    const int lane = threadIdx.x & 31;
    const long long kb = (K + 1) / 2;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < groups; i += (long long)gridDim.x * 8) {
        const long long row = i / ng;
        const long long k0 = (i - row * ng) * group;
        const int cnt = (int)min((long long)group, K - k0);
        const WT* src = w + row * K + k0;
        float lo[2], hi[2], m = 0.0f;  // the weights of the byte pairs this lane writes
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int k = 2 * (lane + 32 * e);
            lo[e] = k < cnt ? src_f32(src + k) : 0.0f;
            hi[e] = k + 1 < cnt ? src_f32(src + k + 1) : 0.0f;
            m = fmaxf(m, fmaxf(fabsf(lo[e]), fabsf(hi[e])));  // fmaxf skips NaN
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t bits = q4_scale_bits(m);
        const float s = bf16_bits_to_f32(bits);
        if (lane == 0) scales[i] = (uint16_t)bits;
        uint8_t* dst = q4 + row * kb + k0 / 2;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int k = 2 * (lane + 32 * e);
            if (k < cnt) dst[k / 2] = (uint8_t)(q4_code(lo[e], s) | (q4_code(hi[e], s) << 4));
        }
    }
}

// Any K, any alignment: a block per output row, a byte (two weights) a thread and step.
template <typename OT>
__global__ void __launch_bounds__(256) q4_dequantize_generic_kernel(OT* __restrict__ out, const uint8_t* __restrict__ q4,
                                                                    const uint16_t* __restrict__ scales,
                                                                    const int* __restrict__ rows, long long R,
                                                                    long long N, long long K, int group)
{
    const long long kb = (K + 1) / 2, ng = (K + group - 1) / group;
    for (long long r = blockIdx.x; r < R; r += gridDim.x) {
        const long long n = rows ? (long long)rows[r] : r;
        const bool in = n >= 0 && n < N;
        OT* o = out + r * K;
        for (long long j = threadIdx.x; j < kb; j += blockDim.x) {
            float a = 0.0f, b = 0.0f;
            if (in) {
                const float s = bf16_bits_to_f32(scales[n * ng + 2 * j / group]);
                const int v = q4[n * kb + j];
                a = (float)((v & 15) - 8) * s;
                b = (float)((v >> 4) - 8) * s;
            }
            store_from_f32<OT>(o + 2 * j, a);
            if (2 * j + 1 < K) store_from_f32<OT>(o + 2 * j + 1, b);
        }
    }
}

template <typename WT>
cudaError_t quantize_typed(const WT* w, size_t N, size_t K, int group, uint8_t* q4, uint16_t* scales, int num_sms,
                           cudaStream_t stream)
{
    const long long ng = (long long)((K + group - 1) / group), groups = ng * (long long)N;
    const long long blocks = std::min<long long>((groups + 7) / 8, (long long)num_sms * 64);
    q4_quantize_generic_kernel<WT><<<(unsigned)blocks, 256, 0, stream>>>(w, q4, scales, groups, (int)ng, (long long)K,
                                                                         group);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename OT>
cudaError_t dequantize_typed(OT* out, const uint8_t* q4, const uint16_t* scales, int group, const int* rows, size_t R,
                             size_t N, size_t K, int num_sms, cudaStream_t stream)
{
    const long long blocks = std::min<long long>((long long)R, (long long)num_sms * 64);
    q4_dequantize_generic_kernel<OT><<<(unsigned)blocks, 256, 0, stream>>>(out, q4, scales, rows, (long long)R,
                                                                           (long long)N, (long long)K, group);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace

cudaError_t launch_q4_quantize(const void* w, int w_bf16, size_t N, size_t K, int group, uint8_t* q4, uint16_t* scales,
                               int num_sms, cudaStream_t stream)
{
    return w_bf16 ? quantize_typed<uint16_t>(static_cast<const uint16_t*>(w), N, K, group, q4, scales, num_sms, stream)
                  : quantize_typed<float>(static_cast<const float*>(w), N, K, group, q4, scales, num_sms, stream);
}

cudaError_t launch_q4_dequantize(void* out, int out_dtype, const uint8_t* q4, const uint16_t* scales, int group,
                                 const int* rows, size_t R, size_t N, size_t K, int num_sms, cudaStream_t stream)
{
    return out_dtype == kF16
               ? dequantize_typed<__half>(static_cast<__half*>(out), q4, scales, group, rows, R, N, K, num_sms, stream)
               : dequantize_typed<float>(static_cast<float*>(out), q4, scales, group, rows, R, N, K, num_sms, stream);
}

}  // namespace b200q8
