// q4_quantize.cu -- 4-bit group quantization of weights (fp32 or bf16) and its inverse.
//
// Per group of `group` consecutive weights of a row: s = bf16(max |w| / 7) with NaN skipped,
// q = round(w / s) (ties to even) within -8..7 (q4_common.cuh).  Deterministic and exact, so the
// codes of a matrix are a function of its values alone.
//
// Both are bound by HBM: the large case of each direction reads or writes 4 bytes a weight.
//
// Dequantization writes q * s for all rows, or for a list of rows: the token lookup of a tied
// embedding / output head that is kept in 4 bits.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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

// Eight consecutive weights, as pairs.
__device__ __forceinline__ void load8(const float* p, float2* v)
{
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
}
__device__ __forceinline__ void load8(const uint16_t* p, float2* v)
{
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}

// Aligned rows of octets (K % 8 == 0): the matrix as one run of octets of weights; kShort: rows end within a
// group, and threads stand for the missing octets, `per_row` runs of octets to a row in all.  A thread takes O
// consecutive octets (16 bytes of bf16 or 32 of fp32 each), neighbouring threads a group, and U such
// runs at a time.  bf16 takes two octets a thread: a group's scale is then worked out by half as many.
// The quotients are IEEE's without a division per weight: with y = 1 / s rounded to nearest, t = w y and the
// exact remainder w - t s, t + (w - t s) y is the correctly rounded w / s (Markstein), in packed
// operations; adding 1.5 * 2^23 then rounds it to an integer, ties to even.  Groups whose 1 / s is no normal
// number and NaN weights take the plain way.
// Bound by HBM for fp32 (18944 x 3584: 44 us, 6.9 TB/s), by HBM and instruction issue for bf16 (37888 x 3584: 56 us);
// rows that end within a group 26316 x 2592 57 us in fp32, 48 in bf16 (the generic kernel: 200).
template <typename WT, int G, int O, int U, bool kShort>
__global__ void __launch_bounds__(256) q4_quantize_flat_kernel(const WT* __restrict__ w, uint32_t* __restrict__ q4,
                                                               uint16_t* __restrict__ scales, long long runs, int per_row, int K)
{
    constexpr int kLanes = G / (8 * O);  // threads of a group
    // Where run r's weights lie, in runs; false: behind its row's end.
    auto find = [&](long long r, long long& at) {
        at = r;
        if (!kShort) return r < runs;
        const long long row = r / per_row;
        const int c = (int)(r - row * per_row), have = K / (8 * O);
        at = row * have + c;
        return r < runs && c < have;
    };
    pdl_wait();
    pdl_launch_dependents();
    const long long base = (long long)blockIdx.x * (256 * U) + threadIdx.x;
    float2 v[U][4 * O];
#pragma unroll
    for (int i = 0; i < U; i++) {
        long long at;
        const bool in = find(base + i * 256, at);
#pragma unroll
        for (int o = 0; o < O; o++)
            if (in)
                load8(w + (at * O + o) * 8, v[i] + 4 * o);
            else
                v[i][4 * o] = v[i][4 * o + 1] = v[i][4 * o + 2] = v[i][4 * o + 3] = make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const long long r = base + i * 256;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 4 * O; j++) m = fmaxf(m, fmaxf(fabsf(v[i][j].x), fabsf(v[i][j].y)));  // fmaxf skips NaN
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const uint32_t bits = q4_scale_bits(m);
        const float s = bf16_bits_to_f32(bits);
        const float inv = s > 1e-30f && s < 1e30f ? __frcp_rn(s) : NAN;
        const float2 y = make_float2(inv, inv), ns = make_float2(-s, -s);
        const float2 round = make_float2(12582912.0f + 8.0f, 12582912.0f + 8.0f);  // + 8: the code
        uint32_t code[O];
        float2 all = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int o = 0; o < O; o++) {
            uint32_t c = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 x = v[i][4 * o + j];
                float2 t = __fmul2_rn(x, y);
                t = __ffma2_rn(__ffma2_rn(t, ns, x), y, t);
                all = __fadd2_rn(all, t);
                t = __fadd2_rn(t, round);
                c += (__float_as_uint(t.x) << (8 * j)) + (__float_as_uint(t.y) << (8 * j + 4));
            }
            // every float's bits are 0x4B400000 + code: take what the upper parts add up to off again
            constexpr uint32_t kUpper = 0x4B400000u * 0x11111111u;
            code[o] = c - kUpper;
        }
        if (!(fabsf(all.x + all.y) <= 1e6f)) {
#pragma unroll
            for (int o = 0; o < O; o++) {
                code[o] = 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    code[o] |= q4_code(v[i][4 * o + j].x, s) << (8 * j) | q4_code(v[i][4 * o + j].y, s) << (8 * j + 4);
            }
        }
        long long at;
        if (find(r, at)) {  // (a group's first octet is there)
            if constexpr (O == 2)
                __stcs(reinterpret_cast<uint2*>(q4) + at, make_uint2(code[0], code[1]));
            else
                __stcs(q4 + at, code[0]);
            if (threadIdx.x % kLanes == 0) scales[r / kLanes] = (uint16_t)bits;
        }
    }
}

// What a thread dequantizes at a time: 16 bytes of output, so that a warp's stores are whole lines.
template <typename OT>
struct Piece;
template <>
struct Piece<float> {
    using Codes = uint16_t;
    static constexpr int kLog2 = 2;  // of its weights
    static __device__ __forceinline__ void store(float* p, uint32_t w, float s)
    {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++)  // 2^23 + code, less 2^23 + 8
            v[j] = (__uint_as_float(((w >> (4 * j)) & 15u) | 0x4B000000u) - 8388616.0f) * s;
        __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    }
};
template <>
struct Piece<__half> {
    using Codes = uint32_t;
    static constexpr int kLog2 = 3;
    static __device__ __forceinline__ void store(__half* p, uint32_t w, float s)
    {
        uint4 r;
        uint32_t* d = &r.x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = (__uint_as_float(((w >> (8 * i)) & 15u) | 0x4B000000u) - 8388616.0f) * s;
            const float b = (__uint_as_float(((w >> (8 * i + 4)) & 15u) | 0x4B000000u) - 8388616.0f) * s;
            const __half2 h = __floats2half2_rn(a, b);
            d[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        __stcs(reinterpret_cast<uint4*>(p), r);
    }
};

// All rows, whole groups, aligned: the matrix as one run of pieces, U of them a thread in flight.
template <typename OT, int U>
__global__ void __launch_bounds__(256) q4_dequantize_flat_kernel(OT* __restrict__ out, const uint8_t* __restrict__ q4,
                                                                 const uint16_t* __restrict__ scales, long long pieces,
                                                                 int group_log2)
{
    using P = Piece<OT>;
    pdl_wait();
    pdl_launch_dependents();
    const auto* codes = reinterpret_cast<const typename P::Codes*>(q4);
    const long long base = (long long)blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t w[U];
    float s[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        const long long o = base + i * 256;
        w[i] = o < pieces ? __ldcs(codes + o) : 0u;
        s[i] = o < pieces ? bf16_bits_to_f32(__ldg(scales + (o >> (group_log2 - P::kLog2)))) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const long long o = base + i * 256;
        if (o < pieces) P::store(out + (o << P::kLog2), w[i], s[i]);
    }
}

// A list of rows (or rows of broken groups), K % 8 == 0, aligned: a row to blockIdx.x, two pieces a thread.
template <typename OT>
__global__ void __launch_bounds__(256) q4_dequantize_rows_kernel(OT* __restrict__ out, const uint8_t* __restrict__ q4,
                                                                 const uint16_t* __restrict__ scales,
                                                                 const int* __restrict__ rows, int N, int pieces,
                                                                 int ng, int group_log2)
{
    using P = Piece<OT>;
    pdl_wait();
    pdl_launch_dependents();
    const long long r = blockIdx.x;
    const int n = rows ? rows[r] : (int)r;
    const bool in = n >= 0 && n < N;
    const auto* codes = reinterpret_cast<const typename P::Codes*>(q4) + (size_t)(in ? n : 0) * pieces;
    const uint16_t* sc = scales + (size_t)(in ? n : 0) * ng;
    for (int o = blockIdx.y * blockDim.x * 2 + threadIdx.x; o < pieces; o += gridDim.y * blockDim.x * 2) {
        const int o2 = o + blockDim.x;
        uint32_t w = 0, w2 = 0;
        float s = 0.0f, s2 = 0.0f;
        if (in) {
            w = __ldg(codes + o);
            s = bf16_bits_to_f32(__ldg(sc + (o >> (group_log2 - P::kLog2))));
            if (o2 < pieces) {
                w2 = __ldg(codes + o2);
                s2 = bf16_bits_to_f32(__ldg(sc + (o2 >> (group_log2 - P::kLog2))));
            }
        } else {
            w = w2 = 0x88888888u;  // zeros, not minus zeros
        }
        P::store(out + ((r * pieces + o) << P::kLog2), w, s);
        if (o2 < pieces) P::store(out + ((r * pieces + o2) << P::kLog2), w2, s2);
    }
}

int log2_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

template <class... P, class... A>
cudaError_t launch_pdl(void (*kern)(P...), dim3 grid, dim3 block, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
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

template <typename WT>
cudaError_t quantize_typed(const WT* w, size_t N, size_t K, int group, uint8_t* q4, uint16_t* scales, int num_sms,
                           cudaStream_t stream)
{
    const long long ng = (long long)((K + group - 1) / group), groups = ng * (long long)N;
    auto flat = [&](auto octets, auto short_rows) {
        constexpr int O = decltype(octets)::value, U = 2;
        constexpr bool kShort = decltype(short_rows)::value;
        const long long per_row = ng * (group / (8 * O)), runs = per_row * (long long)N;
        const dim3 grid((unsigned)((runs + 256 * U - 1) / (256 * U)));
        auto go = [&](auto kern) {
            return launch_pdl(kern, grid, dim3(256), stream, w, reinterpret_cast<uint32_t*>(q4), scales, runs, (int)per_row, (int)K);
        };
        return group == 32   ? go(q4_quantize_flat_kernel<WT, 32, O, U, kShort>)
               : group == 64 ? go(q4_quantize_flat_kernel<WT, 64, O, U, kShort>)
                             : go(q4_quantize_flat_kernel<WT, 128, O, U, kShort>);
    };
    constexpr int O = sizeof(WT) == 2 ? 2 : 1;
    using One = std::integral_constant<int, 1>;
    if (K % 8 == 0 && aligned(w, 16) && aligned(q4, 4 * O)) {
        if (K % group == 0) return flat(std::integral_constant<int, O>(), std::false_type());
        if (O == 2 && K % 16 == 0) return flat(std::integral_constant<int, O>(), std::true_type());
        return flat(One(), std::true_type());
    }
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
    if (K % 8 == 0 && aligned(q4, 4) && aligned(out, 16)) {
        if (!rows && K % group == 0) {
            constexpr int U = sizeof(OT) == 4 ? 8 : 4;
            const long long pieces = (long long)N * (long long)(K >> Piece<OT>::kLog2);
            return launch_pdl(q4_dequantize_flat_kernel<OT, U>, dim3((unsigned)((pieces + 256 * U - 1) / (256 * U))),
                              dim3(256), stream, out, q4, scales, pieces, log2_of(group));
        }
        const int pieces = (int)(K >> Piece<OT>::kLog2);
        const int threads = std::min(256, (pieces + 63) / 64 * 32);
        const dim3 grid((unsigned)R, (unsigned)std::min((pieces + 2 * threads - 1) / (2 * threads), 65535));
        return launch_pdl(q4_dequantize_rows_kernel<OT>, grid, dim3((unsigned)threads), stream, out, q4, scales, rows,
                          (int)N, pieces, (int)((K + group - 1) / group), log2_of(group));
    }
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
