// q4_common.cuh -- the 4-bit group-quantized weight format, shared by its kernels.
//
// w[n, k] = q[n, k] * s[n, k / group]: q an integer in -8..7 held as the code q + 8, s a bf16.
// Row n holds ceil(K / 2) bytes (element 2j in the low, 2j + 1 in the high four bits of byte j; an
// odd row's last high half holds code 8, the value 0) and ceil(K / group) scales (a row's last group
// may be short).  group is 32, 64 or 128, so no byte belongs to two groups.
// q * s has at most 3 + 8 significant bits: exact in fp32, and in fp16 as long as the exponent fits.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200q8 {

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }

// Round to nearest bf16, ties to even; the result's bits.  Not for NaN.
__device__ __forceinline__ uint32_t f32_to_bf16_bits(float v)
{
    const uint32_t u = __float_as_uint(v);
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// The scale of a group whose largest |w| is `absmax`: the bf16 nearest to absmax / 7.  (Rounding the
// fp32 quotient again gives that same bf16: a quotient could only land on a bf16 midpoint m by
// rounding if |absmax - 7m| <= 3.5 fp32 steps of m, but 7m has 12 significant bits and fp32 numbers
// near it lie at least 4 such steps apart, so absmax = 7m, a true tie.)
__device__ __forceinline__ uint32_t q4_scale_bits(float absmax)
{
    const float s = __fdiv_rn(absmax, 7.0f);
    return s == INFINITY ? 0x7F80u : f32_to_bf16_bits(s);
}

// Code of w under scale s: the integer nearest to w / s (ties to even), within -8..7, plus 8.  The fp32
// quotient decides as the exact one does: for a half integer h, h * s has at most 13 significant
// bits, and w / s can round to h only if w lies within less than one fp32 step of h * s, so w = h * s.
// A group of zeros (s = 0) and NaN weights give the value 0.
__device__ __forceinline__ uint32_t q4_code(float w, float s)
{
    const float r = rintf(__fdiv_rn(w, s));
    const int q = (int)fminf(fmaxf(r, -8.0f), 7.0f);  // fmaxf(NaN, -8) = -8
    return (s > 0.0f && r == r) ? (uint32_t)(q + 8) : 8u;
}

}  // namespace b200q8
