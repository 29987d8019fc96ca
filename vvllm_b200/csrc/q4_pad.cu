// q4_pad.cu -- 4-bit weights and tokens copied into rows that the fast kernels take: K a multiple of 32, rows
// and pointers aligned to 16 bytes.  Behind a row's end come zeros (code 8).
//
// Costs a read and a write of what is copied, bound by HBM, which the fast kernels win back: 37888 x 3583, one token
// 43 us against the generic kernel's 281, eight tokens 46 against 481; 512 tokens by 3584 x 3583 43 against 4611.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace b200q8 {

namespace {

constexpr int kThreads = 256;

// A 16-byte piece of a padded row to a thread and step; `pieces` of them to a row.  The row's bytes lie at
// any address: five aligned words are shifted into four, of which those not wholly inside the matrix are
// put together from bytes.
__global__ void __launch_bounds__(kThreads) q4_pad_rows_kernel(uint4* __restrict__ dst, const uint8_t* __restrict__ src, long long N,
                                                               long long kb, int pieces)
{
    pdl_wait();
    pdl_launch_dependents();
    const uintptr_t begin = reinterpret_cast<uintptr_t>(src), end = begin + (size_t)N * kb;
    const long long total = N * pieces;
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
        const long long n = i / pieces;
        const int j = (int)(i - n * pieces);
        const uintptr_t p = begin + n * kb + 16 * (long long)j, q = p & ~(uintptr_t)3;
        uint32_t w[5];
#pragma unroll
        for (int k = 0; k < 5; k++) {
            const uintptr_t a = q + 4 * k;
            if (a >= begin && a + 4 <= end) {
                w[k] = __ldg(reinterpret_cast<const uint32_t*>(a));
            } else {
                w[k] = 0;
                for (int b = 0; b < 4; b++)
                    if (a + b >= begin && a + b < end) w[k] |= (uint32_t) * reinterpret_cast<const uint8_t*>(a + b) << (8 * b);
            }
        }
        const int left = (int)min((long long)16, kb - 16 * (long long)j);  // bytes of the row
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int have = left - 4 * k;  // of this word's bytes
            const uint32_t keep = have >= 4 ? 0xFFFFFFFFu : have <= 0 ? 0u : (1u << (8 * have)) - 1u;
            o[k] = (__funnelshift_r(w[k], w[k + 1], 8 * (int)(p & 3)) & keep) | (0x88888888u & ~keep);
        }
        dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// [M, K] -> [M, Kp], Kp - K zeros behind every row; T an integer of the elements' size.
template <typename T>
__global__ void __launch_bounds__(kThreads) q4_pad_tokens_kernel(T* __restrict__ dst, const T* __restrict__ src, long long total,
                                                                 long long K, int Kp)
{
    pdl_wait();
    pdl_launch_dependents();
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
        const long long m = i / Kp, k = i - m * Kp;
        dst[i] = k < K ? src[m * K + k] : (T)0;
    }
}

template <class... P, class... A>
cudaError_t launch(void (*kern)(P...), long long work, int num_sms, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<long long>((work + kThreads - 1) / kThreads, (long long)num_sms * 16));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e == cudaSuccess) note_launch();
    return e;
}

size_t padded(size_t K) { return (K + 31) / 32 * 32; }
bool weights_fit(const Q4Args& a) { return a.K % 32 == 0 && (uintptr_t)a.q4 % 16 == 0; }
bool tokens_fit(const Q4Args& a) { return a.K % 32 == 0 && (uintptr_t)a.x % 16 == 0; }
size_t token_bytes(const Q4Args& a) { return a.in_dtype == kF16 ? 2 : 4; }

}  // namespace

size_t q4_pad_bytes(const Q4Args& a)
{
    const size_t kp = padded(a.K);
    return (weights_fit(a) ? 0 : a.N * kp / 2) + (tokens_fit(a) ? 0 : a.M * kp * token_bytes(a));
}

cudaError_t launch_q4_pad(Q4Args* a, unsigned char* to, int num_sms, cudaStream_t stream)
{
    const Q4Args s = *a;
    const size_t kp = padded(s.K);
    if (kp > (size_t)INT32_MAX) return cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess;
    if (!weights_fit(s)) {
        const int pieces = (int)(kp / 32);
        e = launch(q4_pad_rows_kernel, (long long)s.N * pieces, num_sms, stream, reinterpret_cast<uint4*>(to), s.q4, (long long)s.N,
                   (long long)(s.K + 1) / 2, pieces);
        a->q4 = to;
        to += s.N * kp / 2;
    }
    if (e == cudaSuccess && !tokens_fit(s)) {
        const long long total = (long long)(s.M * kp);
        if (s.in_dtype == kF16)
            e = launch(q4_pad_tokens_kernel<uint16_t>, total, num_sms, stream, reinterpret_cast<uint16_t*>(to),
                       static_cast<const uint16_t*>(s.x), total, (long long)s.K, (int)kp);
        else
            e = launch(q4_pad_tokens_kernel<uint32_t>, total, num_sms, stream, reinterpret_cast<uint32_t*>(to),
                       static_cast<const uint32_t*>(s.x), total, (long long)s.K, (int)kp);
        a->x = to;
    }
    a->K = kp;  // as many groups: a group is a multiple of 32
    return e;
}

}  // namespace b200q8
