// q4_gemv.cu -- 4-bit group-quantized weights times a few tokens.
//
// out[m, n] = sum_k x[m, k] * q[n, k] * s[n, k / group] (+ bias[n]) (+ res[m, n]), sums in fp32.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "q4_common.cuh"

namespace b200q8 {

namespace {

// v = acc (+ bias) (+ residual), rounded once to the output type.
template <typename OT>
__device__ __forceinline__ void q4_store(OT* out, const OT* res, float acc, const float* bias, long long n)
{
    float v = acc;
    if (bias) v = __fadd_rn(v, bias[n]);
    if (res) v = __fadd_rn(v, load_as_f32<OT>(res));
    store_from_f32<OT>(out, v);
}

// Any K, any alignment: a warp per weight row and up to 8 tokens, two weights a lane and step.
constexpr int kGenericTokens = 8;
template <typename IT, typename OT>
__global__ void __launch_bounds__(256) q4_linear_generic_kernel(const Q4Args a)
{
    const int lane = threadIdx.x & 31;
    const long long n = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= (long long)a.N) return;
    const long long K = (long long)a.K, kb = (K + 1) / 2, ng = (K + a.group - 1) / a.group;
    const uint8_t* w = a.q4 + n * kb;
    const uint16_t* sc = a.scales + n * ng;
    for (long long m0 = (long long)blockIdx.y * kGenericTokens; m0 < (long long)a.M;
         m0 += (long long)gridDim.y * kGenericTokens) {
        const int mt = (int)min((long long)kGenericTokens, (long long)a.M - m0);
        const IT* x = static_cast<const IT*>(a.x) + m0 * K;
        float acc[kGenericTokens] = {};
        for (long long j = lane; j < kb; j += 32) {
            const float s = bf16_bits_to_f32(sc[2 * j / a.group]);
            const int v = w[j];
            const float w0 = (float)((v & 15) - 8) * s, w1 = (float)((v >> 4) - 8) * s;  // exact
            const bool two = 2 * j + 1 < K;
#pragma unroll
            for (int m = 0; m < kGenericTokens; m++)
                if (m < mt) {
                    acc[m] = fmaf(w0, load_as_f32<IT>(x + m * K + 2 * j), acc[m]);
                    if (two) acc[m] = fmaf(w1, load_as_f32<IT>(x + m * K + 2 * j + 1), acc[m]);
                }
        }
#pragma unroll
        for (int m = 0; m < kGenericTokens; m++) {
            const float v = warp_sum(acc[m]);
            if (m < mt && lane == m) {
                const long long o = (m0 + m) * (long long)a.N + n;
                q4_store<OT>(static_cast<OT*>(a.out) + o, a.res ? static_cast<const OT*>(a.res) + o : nullptr, v, a.bias, n);
            }
        }
    }
}

template <typename IT, typename OT>
cudaError_t launch_generic(const Q4Args& a, cudaStream_t stream)
{
    const dim3 grid((unsigned)((a.N + 7) / 8),
                    (unsigned)std::min<size_t>((a.M + kGenericTokens - 1) / kGenericTokens, 65535));
    q4_linear_generic_kernel<IT, OT><<<grid, 256, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace

cudaError_t launch_q4_linear_generic(const Q4Args& a, cudaStream_t stream)
{
    if (a.in_dtype == kF16)
        return a.out_dtype == kF16 ? launch_generic<__half, __half>(a, stream) : launch_generic<__half, float>(a, stream);
    return a.out_dtype == kF16 ? launch_generic<float, __half>(a, stream) : launch_generic<float, float>(a, stream);
}

}  // namespace b200q8
