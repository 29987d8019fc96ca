// q4_gemv.cu -- 4-bit group-quantized weights times a few tokens.
//
// out[m, n] = sum_k x[m, k] * q[n, k] * s[n, k / group] (+ bias[n]) (+ res[m, n]), sums in fp32.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "q4_common.cuh"
#include "tc_utils.cuh"
#include "tmap.cuh"

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


// ----------------------------------------------------------------------------------------------
// Streaming kernel: K % 32 == 0, aligned pointers, up to 16 tokens (8 in fp32) to a CTA and pass over the weights.
//
// Three to sixteen fp16 tokens: the codes become the integers q in fp16 (nine operations per eight), and
// mma.sync m16n8k16 multiplies them with the tokens as they are; products are exact, the tensor core sums a
// group's, and the group's sum times its scale is added to the row's in fp32.
//
// One or two tokens, and fp32 tokens: exact integer products.  A token's 128 consecutive elements ("chunk")
// become integers X = rint(x * 2^(22 - e)), 2^e above the chunk's largest |x|, and X three signed bytes
// X = 65536 X2 + 256 X1 + X0: three columns of the product.  The codes become bytes 16 q with three
// integer operations per eight (one shift, two and-xor).  So mma.sync m16n8k32 (s8) sums 16 q * Xd
// of a group exactly, and in fp32 every group's sum is multiplied by the group's scale and the
// chunk's power of two and added to the row's.  What is rounded: an element, by at most 2^-22 of its
// chunk's largest (fp16 tokens are exact down to 2^-11 of it), and the fp32 sums, once a group.  A chunk that
// holds an infinity or NaN is summed directly instead.  Chunks below 2^-100 count as below 2^-100.
// It shows beside activations thousands of times their neighbours', in rows of weights that are 0 there: beside 1000
// the neighbours are held in steps of 2.4e-4.  A fourth byte (2^-30) takes that away and costs, in us: 37888 x 3584
// one token 13.4 -> 13.7, 4096 x 14336 one 13.0 -> 14.1, 3584 x 18944 eight fp32 ones 24.8 -> 33.1, 64 by 3584 x 3584
// 24.3 -> 29.6; beside what four bits round off the weights it is not worth that.
//
// Why both: bytes take a third of the unpacking and half the products, which decides for one token (37888 x 3584:
// in fp16 17.9 us, here 13.4); but each token is three columns and has to be taken apart in every CTA, which
// decides from three on (8 tokens: in bytes 22.5 us, in fp16 17.1; 3584 x 3584 9.3 and 5.7).  Why not
// tcgen05: its operands would have to be written back to shared or tensor memory, twice to four times
// what was read; at 8 cycles a product, mma.sync is within what HBM allows (about 44 cycles for 16 x 32
// weights) to 16 tokens.
//
// Bound by HBM (half a byte a weight) for one and two tokens once there are megabytes to stream: 152064 x 3584
// at 46 us, 6.1 TB/s; 37888 x 3584 at 13.4 us, of which 3 are start and tokens.  With more, by latencies: at 8 tokens no
// unit is full (issue slots 59 %, ALU 50 %, tensor pipe 23 %), and 16 warps an SM do not cover the chain from a
// box over its unpacking to its products: 8 tokens, 152064 x 3584 64 us, 37888 x 3584 17; 16 tokens 93 and 24.5; three
// and eight fp32 ones 24 and 26.5 (three products a token's byte); with long K also by
// the tokens' way into shared memory: 3584 x 18944 12 us at one, 17.5 at eight.
//
// Work: a tile is 16 rows; an item is a tile's next 256 or 512 of K.  `wk` warps share a tile (item ch
// goes to warp ch mod wk) and add their sums through shared memory in warp order; a CTA of 8 or 16
// warps has warps / wk such groups, each going through its own tiles.  Every warp has its own ring of
// TMA copies ([16 rows x 128 bytes], 128-byte swizzle), running ahead across tile ends.  Tokens are put
// into shared memory once per CTA.  Where a tile's K is split over a cluster's CTAs (few tiles, or
// tokens too long for one CTA's shared memory), rank 0 adds the CTAs' sums from its shared memory in
// rank order.  No workspace, no atomics: the result does not depend on timing.
//
// Which k a lane holds: within a group, lane t of a row's four takes group / 4 consecutive weights,
// one shared load of 4, 8 or 16 bytes; a sum over k is in whatever order, as the tokens are laid
// out to match.  Fragment row g is tile row rho(g), the bit reversal of g: with it the rows that one
// phase of such a load touches differ in the swizzle's chunk, so there are no bank conflicts.
//
// A copy's wait is bounded: when it runs out the error word is set, the warp goes on without
// waiting or copying (its outputs are invalid), and before it ends waits, bounded again, for the
// copies it has in flight.
constexpr int kMaxWarps = 16;
constexpr int kBoxK = 256;  // K of one copied box: 128 bytes of each of 16 rows
constexpr int kBoxBytes = 16 * 128;
constexpr int kMaxStages = 4;
constexpr int kMaxTokens = 16;      // of one launch: fp16 in halves,
constexpr int kMaxDigitTokens = 8;  // in digits
constexpr uint64_t kWaitNs = 4000000000ull;  // far above any legitimate wait

struct StreamParams {
    Q4Args a;
    int M;            // tokens of this launch, `tokens` of them to blockIdx.y
    int tokens;
    int wk, wk_log2;  // warps per tile
    int stages;       // items in flight per warp
    int nch;          // items per row
    int per;          // items of one cluster rank
    int tiles;
};

__device__ int g_q4_error;  // bit 0: a bounded wait ran out

// Shared loads that the compiler may schedule: an address from `fence` keeps them behind a wait, and
// `fence` on what was computed from them keeps them before the stage is given back.
template <int W>
__device__ __forceinline__ void lds(uint32_t a, uint32_t (&w)[W])
{
    static_assert(W == 1 || W == 2 || W == 4, "4, 8 or 16 bytes");
    if constexpr (W == 1)
        asm("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
    else if constexpr (W == 2)
        asm("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    else
        asm("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
}
// N words from global memory in one load.
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[1]) { w[0] = __ldg(reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[2])
{
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
}
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[4])
{
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
}
__device__ __forceinline__ void fence(uint32_t& v) { asm volatile("" : "+r"(v)::"memory"); }
__device__ __forceinline__ void fence(float& v) { asm volatile("" : "+f"(v)::"memory"); }

// The eight codes of a word as bytes 16 q: elements 0, 2, 4, 6 and 1, 3, 5, 7.  (a & mask) ^ flip with the
// flip turning q + 8 into the two's complement of q, in the upper half of each byte.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t& even, uint32_t& odd)
{
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(even) : "r"(w << 4), "r"(0xF0F0F0F0u), "r"(0x80808080u));
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(odd) : "r"(w), "r"(0xF0F0F0F0u), "r"(0x80808080u));
}

// d += A (16 x 32, s8, rows) * B (32 x 8, s8, columns); with kFirst d = `start` in every element + A * B
template <bool kFirst>
__device__ __forceinline__ void mma16832(int (&d)[4], int start, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1)
{
    if constexpr (kFirst)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(start));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The eight codes of a word as the integers q in fp16: elements (0, 4), (1, 5), (2, 6), (3, 7).  A code in the low
// bits of 1024.0 is 1024 + code, one four bits up 1024 + 16 code; one packed fma leaves q.  (Converting small integers
// under an exponent: Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022.)
__device__ __forceinline__ void unpack8_halves(uint32_t w, uint32_t (&h)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = i < 2 ? w : w >> 8;
        if (i & 1) {
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(h[i]) : "r"(v), "r"(0x00F000F0u), "r"(0x64006400u));
            asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(h[i]) : "r"(0x2C002C00u), "r"(0xD480D480u));  // / 16 - 72
        } else {
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(h[i]) : "r"(v), "r"(0x000F000Fu), "r"(0x64006400u));
            asm("add.rn.f16x2 %0, %0, %1;" : "+r"(h[i]) : "r"(0xE408E408u));  // - 1032
        }
    }
}

// d += A (16 x 16, fp16, rows) * B (16 x 8, fp16, columns), or with kFirst d = A * B; fp32 sums
template <bool kFirst>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    if constexpr (kFirst)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The sums start at the bit pattern of 1.5 * 2^23: read as a float they are that plus the sum, exact
// while |sum| < 2^22 (a group's is at most 128 * 128 * 128 = 2^21).
constexpr int kMagicBits = 0x4B400000;
constexpr float kMagic = 12582912.0f;

// The sums of a fragment's columns 2t and 2t + 1 in row `i`.
__device__ __forceinline__ float2 tile_value(const int (&d)[4], int i)
{
    return __fadd2_rn(make_float2(__int_as_float(d[2 * i]), __int_as_float(d[2 * i + 1])), make_float2(-kMagic, -kMagic));
}

// Shared memory distance of two columns of `blocks` 32-blocks, of bytes (two blocks to 64 bytes) or fp16 (one): an
// odd number of those, so that neighbouring columns' loads fall into different banks.
__host__ __device__ constexpr size_t column_stride(int blocks, bool halves) { return (size_t)((halves ? blocks : blocks / 2) | 1) * 64; }

// Columns of the product.  Up to two tokens: one 8-column tile, token m's byte d (X0, X1, X2) in column
// 3 m + d.  Up to eight: three tiles, token m in column m of tile d.
template <int NT>
__device__ __forceinline__ int column_of(int m, int d, int M)  // where it is stored
{
    return NT == 1 ? 3 * m + d : d * M + m;
}

// Tokens m0 .. m0 + M - 1 into shared memory, `blocks` (a multiple of 8) 32-blocks from block0:
//   xs      [column][pair of blocks][quarter t][2 blocks] of 8 bytes: the bytes that lane t multiplies
//           with its word of a block, elements 0 2 4 6 1 3 5 7.  Within a group of W = group / 32 blocks, word
//           w of lane t starts at element (t * W + w) * 8.  Zero behind K.
//   weight  [chunk][8]: what a column's integer (NT == 1; else a token's X) counts, with the 1/16 of the codes' bytes
//   direct  [token][chunk]: 1 if the chunk is summed directly; returns whether this thread saw any
// Half a warp per chunk of 128 elements, eight elements a lane; a few chunks' loads at a time.  `asked` is
// called once the first loads are under way, `arrived` once they are there.
template <int NT, bool kF16, class Asked, class Arrived>
__device__ __forceinline__ bool stage_tokens(unsigned char* xs, float* weight, unsigned char* direct,
                                             const StreamParams& p, int m0, int M, int W, int block0, int blocks, Asked asked, Arrived arrived)
{
    constexpr int U = 5;  // chunks whose loads are in flight
    constexpr int kRaw = kF16 ? 4 : 8;
    const int K = (int)p.a.K, chunks = blocks / 4;
    const size_t cs = column_stride(blocks, false);
    const int u = threadIdx.x & 15;  // word of the chunk
    const int half = threadIdx.x >> 4, halves = blockDim.x >> 4;
    const int o = u & (4 * W - 1), ub = u / (4 * W) * W + (o & (W - 1));  // its block in the chunk
    unsigned char* const dst0 = xs + (ub >> 1) * 64 + (o / W) * 16 + (ub & 1) * 8;
    bool any = false, first = true;
    // Rounds: every half warp a chunk of one token, chunks c0 + half.
    for (int m = 0, c0 = 0; m < M;) {
        uint32_t raw[U][kRaw];
        int lm = m, lc = c0;
#pragma unroll
        for (int q = 0; q < U; q++) {
            const int k = block0 * 32 + (lc + half) * 128 + u * 8;
#pragma unroll
            for (int j = 0; j < kRaw; j++) raw[q][j] = 0;
            if (lm < M && lc + half < chunks && k < K) {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p.a.x) +
                                                                  ((size_t)(m0 + lm) * K + k) * (kF16 ? 2 : 4));
#pragma unroll
                for (int j = 0; j < kRaw / 4; j++) {
                    const uint4 r = src[j];
                    raw[q][4 * j] = r.x, raw[q][4 * j + 1] = r.y, raw[q][4 * j + 2] = r.z, raw[q][4 * j + 3] = r.w;
                }
            }
            lc += halves;
            if (lc >= chunks) lc = 0, lm++;
        }
        if (first) asked();
#pragma unroll
        for (int q = 0; q < U; q++) {
            if (m >= M) break;  // uniform in the CTA
            // The largest |x| as bits: above every number for an infinity or NaN.
            float v[8];
            uint32_t top;
            if constexpr (kF16) {
                uint32_t h = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(h) : "r"(raw[q][j] & 0x7FFF7FFFu));
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw[q][j]));
                    v[2 * j] = f.x, v[2 * j + 1] = f.y;
                }
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                top = max(__float_as_uint(f.x), __float_as_uint(f.y));
            } else {
                top = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[j] = __uint_as_float(raw[q][j]);
                    top = max(top, raw[q][j] & 0x7FFFFFFFu);
                }
            }
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (first) arrived();
            first = false;
            const bool bad = top >= 0x7F800000u;
            const int e = max((int)(top >> 23) - 126, -100);  // |x| < 2^e
            const float up = __uint_as_float((uint32_t)(22 - e + 127) << 23);
            // X in the low bits of x * up + 1.5 * 2^23; with 128 added to each byte, the bytes are the signed
            // digits with their top bit flipped.
            uint32_t y[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                y[j] = __float_as_uint(fmaf(v[j], up, kMagic)) + (0x00808080u - (uint32_t)kMagicBits);
            if (bad)
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = 0x00808080u;
            const int c = c0 + half;
            if (c < chunks) {
                unsigned char* dst = dst0 + c * 128;
#pragma unroll
                for (int n = 0; n < 3; n++) {
                    uint32_t d[2];  // the digit of the even and the odd elements
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t lo = __byte_perm(y[h], y[2 + h], n == 2 ? 0x0062 : 0x5140);
                        const uint32_t hi = __byte_perm(y[4 + h], y[6 + h], n == 2 ? 0x0062 : 0x5140);
                        d[h] = __byte_perm(lo, hi, n == 1 ? 0x7632 : 0x5410) ^ 0x80808080u;
                    }
                    *reinterpret_cast<uint2*>(dst + column_of<NT>(m, n, M) * cs) = make_uint2(d[0], d[1]);
                }
                if (u < (NT == 1 ? 3 : 1))
                    weight[c * 8 + (NT == 1 ? 3 * m + u : m)] = __uint_as_float((uint32_t)(e - 22 - 4 + 8 * u + 127) << 23);
                if (u == 3) direct[m * chunks + c] = bad;
                any |= bad;
            }
            c0 += halves;
            if (c0 >= chunks) c0 = 0, m++;
        }
    }
    return any;
}

// fp16 tokens as they are: [column m][block][quarter t] of eight, elements 0 4 1 5 2 6 3 7 of the word that lane t
// multiplies with its word of the block (the words in the order above).  Zero behind K.
template <class Asked, class Arrived>
__device__ __forceinline__ void stage_halves(unsigned char* xs, const StreamParams& p, int m0, int M, int W, int block0, int blocks, Asked asked,
                                             Arrived arrived)
{
    constexpr int U = 8;  // chunks whose loads are in flight
    const int K = (int)p.a.K, chunks = blocks / 4;
    const size_t cs = column_stride(blocks, true);
    const int u = threadIdx.x & 15, half = threadIdx.x >> 4, halves = blockDim.x >> 4;
    const int o = u & (4 * W - 1), ub = u / (4 * W) * W + (o & (W - 1));
    unsigned char* const dst0 = xs + ub * 64 + (o / W) * 16;
    bool first = true;
    for (int m = 0, c0 = 0; m < M;) {
        uint4 raw[U];
        int lm = m, lc = c0;
#pragma unroll
        for (int q = 0; q < U; q++) {
            const int k = block0 * 32 + (lc + half) * 128 + u * 8;
            raw[q] = make_uint4(0, 0, 0, 0);
            if (lm < M && lc + half < chunks && k < K)
                raw[q] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.a.x) + (size_t)(m0 + lm) * K + k);
            lc += halves;
            if (lc >= chunks) lc = 0, lm++;
        }
        if (first) asked();
#pragma unroll
        for (int q = 0; q < U; q++) {
            if (m >= M) break;  // uniform in the CTA
            const uint4 r = raw[q];
            const uint4 v = make_uint4(__byte_perm(r.x, r.z, 0x5410), __byte_perm(r.x, r.z, 0x7632),
                                       __byte_perm(r.y, r.w, 0x5410), __byte_perm(r.y, r.w, 0x7632));
            if (first) arrived();
            first = false;
            const int c = c0 + half;
            if (c < chunks) *reinterpret_cast<uint4*>(dst0 + c * 256 + m * cs) = v;
            c0 += halves;
            if (c0 >= chunks) c0 = 0, m++;
        }
    }
}

// A warp adds to sums[r], r < 16, token m's products with rows tile * 16 + r over 128-chunk c, as the formula
// reads: what infinities and NaN need.
__device__ __noinline__ void direct_chunk(const Q4Args& a, float* sums, int tile, int m, int c)
{
    const int lane = threadIdx.x & 31;
    const size_t K = a.K, ng = (K + a.group - 1) / a.group;
    for (int r = 0; r < 16; r++) {
        const size_t n = (size_t)tile * 16 + r;
        if (n >= a.N) break;
        float v = 0.0f;
        for (int j = lane; j < 64; j += 32) {
            const size_t k = (size_t)c * 128 + 2 * j;
            if (k >= K) break;
            const float s = bf16_bits_to_f32(a.scales[n * ng + k / a.group]);
            const int code = a.q4[(n * K + k) / 2];
            const size_t i = (size_t)m * K + k;
            const float x0 = a.in_dtype == kF16 ? __half2float(static_cast<const __half*>(a.x)[i])
                                                : static_cast<const float*>(a.x)[i];
            const float x1 = a.in_dtype == kF16 ? __half2float(static_cast<const __half*>(a.x)[i + 1])
                                                : static_cast<const float*>(a.x)[i + 1];
            v = fmaf((float)((code & 15) - 8) * s, x0, v);
            v = fmaf((float)((code >> 4) - 8) * s, x1, v);
        }
        v = warp_sum(v);
        if (lane == 0) sums[r] += v;
    }
    __syncwarp();
}

template <int NT, int IB, bool kHalves>
struct StreamCfg {
    static constexpr int kItemBytes = IB * kBoxBytes;
    static constexpr int kChunks = IB * kBoxK / 128;  // 128-chunks of an item
    static constexpr int kCols = kHalves ? 0 : 8;     // columns kept in `weight`: NT == 1 the tile's, else the tokens
    static constexpr int kChunkBytes = kHalves ? 256 : 128;  // of a column
    static constexpr int kOut = kHalves ? NT : 1;            // eights of tokens in a lane's sums
    static constexpr int kSums = (kHalves ? 8 * NT : NT == 1 ? 2 : 8) * 16;  // a tile's outputs: [token][row]
    // Two buffers of sums, read while the next tile's are written, where warps or CTAs share a tile.
    static constexpr int red_bufs(int wk, int cluster) { return wk == 1 && cluster == 1 ? 1 : 2; }
    static size_t smem(int warps, int stages, int M, int per, int cluster, int wk)
    {
        const int chunks = per * kChunks;
        return 1024 + (size_t)warps * stages * kItemBytes + warps * kMaxStages * 8 +
               (kHalves ? 1 : 3) * M * column_stride(chunks * 4, kHalves) + (size_t)chunks * kCols * 4 +
               (size_t)red_bufs(wk, cluster) * warps * kSums * 4 +
               (cluster > 1 ? (size_t)2 * cluster * (warps / wk) * kSums * 4 : 0) + (kHalves ? 0 : (size_t)M * chunks);
    }
};

// kHalves false: the tokens' digits in NT = 1 (up to two tokens) or 3 (up to eight) tiles of eight columns; true: up to
// 8 NT fp16 tokens as they are.
template <int NT, int G, int IB, bool kHalves>
__global__ void __launch_bounds__(kMaxWarps * 32, 1)
    q4_stream_kernel(const __grid_constant__ CUtensorMap tmW, const StreamParams p)
{
    using C = StreamCfg<NT, IB, kHalves>;
    constexpr int kItemBytes = C::kItemBytes;
    constexpr int W = G / 32;   // words a lane holds of a group; 32-blocks of a group
    constexpr int GC = 128 / G;  // groups of a chunk
    constexpr int kBoxGroups = kBoxK / G;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int csize = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warps = blockDim.x >> 5;
    const int m0 = (int)blockIdx.y * p.tokens, M = min(p.tokens, p.M - m0);  // this CTA's tokens
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) &
                                                           ~static_cast<uintptr_t>(1023));
    const int ch0 = rank * p.per, ch1 = min(p.nch, ch0 + p.per);  // items of a row that this CTA takes
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)warps * p.stages * kItemBytes);
    unsigned char* xs = reinterpret_cast<unsigned char*>(bars + warps * kMaxStages);
    const int xchunks = p.per * C::kChunks;
    const size_t cs = column_stride(xchunks * 4, kHalves);
    float* weight = reinterpret_cast<float*>(xs + (kHalves ? 1 : 3) * M * cs);
    float* red = weight + xchunks * C::kCols;         // [buffer][warp][tile's outputs]
    float* cbuf = red + C::red_bufs(p.wk, csize) * warps * C::kSums;  // [2][rank][group][tile's outputs] of a cluster's CTAs (in rank 0)
    unsigned char* direct = reinterpret_cast<unsigned char*>(cbuf + (csize > 1 ? 2 * csize * (warps >> p.wk_log2) * C::kSums : 0));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int row = ((g & 1) << 2) | (g & 2) | (g >> 2);  // rho(g); the fragment's other row is row + 8
    const int wk = p.wk, kw = warp & (wk - 1);
    const int group = warp >> p.wk_log2, groups = warps >> p.wk_log2;
    const int tbase = ((int)blockIdx.x / csize) * groups, tile0 = tbase + group;
    const int tstep = ((int)gridDim.x / csize) * groups;
    const int N = (int)p.a.N, K = (int)p.a.K;
    const int ng = (K + G - 1) / G;

    // ---- copies: the warp's items in order, (tile, ch) with ch = ch0 + kw, + wk, ...
    const uint32_t ring = tc::smem_u32(smem) + warp * p.stages * kItemBytes;
    const uint32_t bar0 = tc::smem_u32(bars + warp * kMaxStages);
    const bool busy = ch0 + kw < ch1;  // there are items for this warp
    int itile = busy ? tile0 : p.tiles, ich = ch0 + kw, inflight = 0;
    auto advance = [&]() {
        ich += wk;
        if (ich >= ch1) {
            ich = ch0 + kw;
            itile += tstep;
        }
    };
    // A tile's scales, 16 rows' worth and contiguous, into L2 ahead of their loads.
    auto prefetch_scales = [&](int tile) {
        const size_t off = (size_t)tile * 16 * ng;
        const uint32_t bytes = (uint32_t)(min(16, N - tile * 16) * ng * 2) & ~15u;
        if (bytes && ((uintptr_t)p.a.scales & 15) == 0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.a.scales + off), "r"(bytes) : "memory");
    };
    if (lane == 0) {
        for (int i = 0; i < p.stages; i++) tc::mbar_init(bar0 + 8 * i, 1);
        tc::fence_mbar_init();
        tc::prefetch_tensormap(&tmW);
        // While the kernel before ends: this warp's first item into L2.  (Into L2 only, where it stays
        // coherent: the kernel before may have written the weights themselves.)
        if (kw == 0 && tile0 < p.tiles) prefetch_scales(tile0);
        if (itile < p.tiles)
            for (int b = 0; b < IB; b++) tc::tma_prefetch_l2_2d(&tmW, (ich * IB + b) * 128, itile * 16);
    }
    pdl_wait();
    pdl_launch_dependents();
    const uint64_t policy = gridDim.y == 1 ? tc::l2_policy_evict_first() : tc::l2_policy_evict_normal();
    auto load_item = [&](int stage) {
        tc::mbar_arrive_expect_tx(bar0 + 8 * stage, kItemBytes);
#pragma unroll
        for (int b = 0; b < IB; b++)  // behind a row's end or the last row: zeros
            tc::tma_load_2d_hint(ring + stage * kItemBytes + b * kBoxBytes, &tmW, (ich * IB + b) * 128, itile * 16,
                                 bar0 + 8 * stage, policy);
    };
    // Scales, two to a word, of the item about to be multiplied; those of the next (with items of one box, of
    // the two next) are loaded meanwhile: a box takes less than a load from L2.
    constexpr int kSW = kBoxGroups / 2;
    struct Scales {
        uint32_t a[IB][kSW], b[IB][kSW];  // the fragment's two rows
    };
    int stile = busy ? tile0 : p.tiles, sch = ch0 + kw;  // the item whose scales are loaded next
    const uint16_t* sp = nullptr;
    size_t srow = 0;  // from the first row's scales to the other's
    const bool swide = ng % kBoxGroups == 0 && ((uintptr_t)p.a.scales & (2 * kBoxGroups - 1)) == 0;  // one load a row and box
    auto load_scales = [&](Scales& s) {
        if (stile >= p.tiles) return;
        if (sch == ch0 + kw) {
            const int n0 = min(stile * 16 + row, N - 1), n1 = min(stile * 16 + row + 8, N - 1);
            sp = p.a.scales + (size_t)n0 * ng + sch * IB * kBoxGroups;
            srow = (size_t)(n1 - n0) * ng;
        }
        const int left = ng - sch * IB * kBoxGroups;  // groups from here to the row's end
#pragma unroll
        for (int b = 0; b < IB; b++) {
            if (swide) {
                if (b * kBoxGroups < left) {
                    load_words(sp + b * kBoxGroups, s.a[b]);
                    load_words(sp + srow + b * kBoxGroups, s.b[b]);
                } else {
#pragma unroll
                    for (int i = 0; i < kSW; i++) s.a[b][i] = s.b[b][i] = 0;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kBoxGroups; i++) {
                    const int j = b * kBoxGroups + i;
                    const bool in = j < left;  // a row's last box may be short
                    const uint32_t x = in ? (uint32_t)__ldg(sp + j) : 0u, y = in ? (uint32_t)__ldg(sp + srow + j) : 0u;
                    s.a[b][i / 2] = i & 1 ? s.a[b][i / 2] | x << 16 : x;
                    s.b[b][i / 2] = i & 1 ? s.b[b][i / 2] | y << 16 : y;
                }
            }
        }
        sch += wk;
        sp += wk * IB * kBoxGroups;
        if (sch >= ch1) {
            sch = ch0 + kw;
            stile += tstep;
        }
    };
    Scales sc{}, sc_next{};

    // The tokens' loads go first, then one item a warp: behind more they would wait for megabytes to pass (all of
    // the ring first: 37888 x 3584, one token, 14.0 us instead of 13.4; 3584 x 18944 13.2, 12.2).  Once they are
    // there the ring is filled, before they are converted.
    auto asked = [&]() {
        if (lane == 0 && itile < p.tiles) {
            load_item(inflight++);
            advance();
        }
        load_scales(sc);
        if (IB == 1) load_scales(sc_next);
    };
    auto arrived = [&]() {
        if (lane == 0)
            for (; inflight < p.stages && itile < p.tiles; inflight++, advance()) load_item(inflight);
    };
    bool any_direct = false;
    if constexpr (kHalves) {
        stage_halves(xs, p, m0, M, W, ch0 * C::kChunks * 4, xchunks * 4, asked, arrived);
        __syncthreads();
    } else {
        const int block0 = ch0 * C::kChunks * 4, blocks = xchunks * 4;
        any_direct = __syncthreads_or(p.a.in_dtype == kF16
                                          ? stage_tokens<NT, true>(xs, weight, direct, p, m0, M, W, block0, blocks, asked, arrived)
                                          : stage_tokens<NT, false>(xs, weight, direct, p, m0, M, W, block0, blocks, asked, arrived));
    }
    if (csize > 1) cluster.sync();  // every rank runs before rank 0's memory is stored to

    uint32_t xoff[NT];  // this lane's column of each 8-column tile (lanes behind the last column repeat it)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
        xoff[nt] = tc::smem_u32(xs) + t * 16 +
                   (uint32_t)((kHalves   ? min(nt * 8 + g, M - 1)
                               : NT == 1 ? min(g, 3 * M - 1)
                                         : nt * M + min(g, M - 1)) * cs);
    // The lane's words of group 0 of a box: 16-byte piece ((t * W) / 4) ^ row of its row; another group is an
    // XOR away.
    const uint32_t wlane = row * 128 + ((((t * W) >> 2) ^ row) << 4) + ((t * W) & 3) * 4;

    const int zero = 0;
    bool ok = true;
    int stage = 0, parity = 0;
    uint32_t phase = 0;
    const int rounds = (p.tiles - tbase + tstep - 1) / tstep;  // uniform in a cluster
    for (int it = 0; it < rounds; it++) {
        const int tile = tile0 + it * tstep;
        if (tile >= p.tiles && csize == 1) break;  // a cluster's groups end together, for its barriers
        if (lane == 0 && kw == 0 && tile + tstep < p.tiles) prefetch_scales(tile + tstep);
        // Of rows row and row + 8: columns 2t and 2t + 1, which are tokens where three tiles hold their bytes.
        float2 acc[C::kOut][2];
#pragma unroll
        for (int o = 0; o < C::kOut; o++) acc[o][0] = acc[o][1] = make_float2(0.0f, 0.0f);
        for (int ch = ch0 + kw; ch < ch1 && tile < p.tiles; ch += wk) {
            if (ok) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(bar0 + 8 * stage, phase, &zero, kWaitNs));
                if (!ok && lane == 0) atomicOr(&g_q4_error, 1);
            }
            uint32_t wrow = ring + stage * kItemBytes + wlane;
            fence(wrow);
            uint32_t xitem = (uint32_t)(ch - ch0) * (C::kChunks * C::kChunkBytes);
            const float* wchunk = weight + (ch - ch0) * C::kChunks * C::kCols + 2 * t;
            // Chunks behind K need no care: their codes and tokens are zeros, and so are their scales.
            Scales sc_after = sc;
            load_scales(sc_after);
#pragma unroll
            for (int box = 0; box < IB; box++) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    if constexpr (kHalves) {
#pragma unroll
                        for (int gi = 0; gi < GC; gi++) {
                            uint32_t w0[W], w1[W];
                            lds<W>(wrow ^ (c * 64 + gi * W * 16), w0);
                            lds<W>((wrow ^ (c * 64 + gi * W * 16)) + 1024, w1);
                            float d[NT][4];
#pragma unroll
                            for (int b = 0; b < W; b++) {
                                uint32_t x[NT][4], h0[4], h1[4];
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) lds<4>(xoff[nt] + xitem + c * 256 + (gi * W + b) * 64, x[nt]);
                                unpack8_halves(w0[b], h0);
                                unpack8_halves(w1[b], h1);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    if (b == 0)
                                        mma16816<true>(d[nt], h0[0], h1[0], h0[1], h1[1], x[nt][0], x[nt][1]);
                                    else
                                        mma16816<false>(d[nt], h0[0], h1[0], h0[1], h1[1], x[nt][0], x[nt][1]);
                                    mma16816<false>(d[nt], h0[2], h1[2], h0[3], h1[3], x[nt][2], x[nt][3]);
                                }
                            }
                            const int si = c * GC + gi;
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const uint32_t word = i == 0 ? sc.a[box][si / 2] : sc.b[box][si / 2];
                                const float r = __uint_as_float(si & 1 ? word & 0xFFFF0000u : word << 16);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++)
                                    acc[nt][i] = __ffma2_rn(make_float2(d[nt][2 * i], d[nt][2 * i + 1]), make_float2(r, r), acc[nt][i]);
                            }
                        }
                    } else {
                        uint32_t x[NT][2][4];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            lds<4>(xoff[nt] + xitem + c * 128, x[nt][0]);
                            lds<4>(xoff[nt] + xitem + c * 128 + 64, x[nt][1]);
                        }
                        float2 sum[2];
#pragma unroll
                        for (int gi = 0; gi < GC; gi++) {
                            uint32_t w0[W], w1[W];
                            lds<W>(wrow ^ (c * 64 + gi * W * 16), w0);
                            lds<W>((wrow ^ (c * 64 + gi * W * 16)) + 1024, w1);
                            int d[NT][4];
#pragma unroll
                            for (int b = 0; b < W; b++) {
                                const int blk = gi * W + b;
                                uint32_t a0, a1, a2, a3;
                                unpack8(w0[b], a0, a2);
                                unpack8(w1[b], a1, a3);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    const uint32_t b0 = x[nt][blk >> 1][2 * (blk & 1)], b1 = x[nt][blk >> 1][2 * (blk & 1) + 1];
                                    if (b == 0)
                                        mma16832<true>(d[nt], kMagicBits, a0, a1, a2, a3, b0, b1);
                                    else
                                        mma16832<false>(d[nt], 0, a0, a1, a2, a3, b0, b1);
                                }
                            }
                            const int si = c * GC + gi;
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const uint32_t word = i == 0 ? sc.a[box][si / 2] : sc.b[box][si / 2];
                                const float r = __uint_as_float(si & 1 ? word & 0xFFFF0000u : word << 16);
                                float2 f = tile_value(d[0], i);
                                if constexpr (NT == 3)  // X0 + 256 X1 + 65536 X2
                                    f = __ffma2_rn(__ffma2_rn(tile_value(d[2], i), make_float2(256.0f, 256.0f), tile_value(d[1], i)),
                                                   make_float2(256.0f, 256.0f), f);
                                sum[i] = gi == 0 ? __fmul2_rn(f, make_float2(r, r)) : __ffma2_rn(f, make_float2(r, r), sum[i]);
                            }
                        }
                        const float2 wt = *reinterpret_cast<const float2*>(wchunk + c * C::kCols);
                        acc[0][0] = __ffma2_rn(sum[0], wt, acc[0][0]);
                        acc[0][1] = __ffma2_rn(sum[1], wt, acc[0][1]);
                    }
                }
                wrow += kBoxBytes;
                xitem += 2 * C::kChunkBytes;
                wchunk += 2 * C::kCols;
            }
            sc = IB == 1 ? sc_next : sc_after;
            sc_next = sc_after;
#pragma unroll
            for (int o = 0; o < C::kOut; o++) fence(acc[o][0].x), fence(acc[o][0].y), fence(acc[o][1].x), fence(acc[o][1].y);
            __syncwarp();  // the stage is read
            if (ok) {  // else the ring stays as it is, for the end
                if (lane == 0) {
                    inflight--;
                    if (itile < p.tiles) {
                        load_item(stage);
                        inflight++;
                        advance();
                    }
                }
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        // ---- v[o][i] of rows row (i < 2) and row + 8, tokens 8 o + mt and, but with digits in one tile, + 1
        float v[C::kOut][4];
#pragma unroll
        for (int o = 0; o < C::kOut; o++)
            v[o][0] = acc[o][0].x, v[o][1] = acc[o][0].y, v[o][2] = acc[o][1].x, v[o][3] = acc[o][1].y;
        constexpr bool kOneTile = !kHalves && NT == 1;
        const int mt = kOneTile ? t >> 1 : 2 * t;
        if constexpr (kOneTile) {  // columns 0 1 | 2, 3 | 4 5 of lanes t = 0, 1, 2: a token's three bytes
            const float a = __shfl_down_sync(0xffffffffu, v[0][0], 1), b = __shfl_down_sync(0xffffffffu, v[0][2], 1);
            const float c = __shfl_up_sync(0xffffffffu, v[0][1], 1), d = __shfl_up_sync(0xffffffffu, v[0][3], 1);
            v[0][0] = t == 0 ? v[0][0] + v[0][1] + a : c + v[0][0] + v[0][1];
            v[0][2] = t == 0 ? v[0][2] + v[0][3] + b : d + v[0][2] + v[0][3];
        }
        auto mine = [&](int o, int i) {  // whether v[o][i] is an output's sum
            return kOneTile ? (t & 1) == 0 && (i & 1) == 0 && mt < M : 8 * o + mt + (i & 1) < M;
        };
        auto put = [&](int m, int r, float y) {
            const long long n = (long long)tile * 16 + r;
            if (n >= N) return;
            const long long o = (long long)(m0 + m) * N + n;
            if (p.a.out_dtype == kF16)
                q4_store<__half>(static_cast<__half*>(p.a.out) + o,
                                 p.a.res ? static_cast<const __half*>(p.a.res) + o : nullptr, y, p.a.bias, n);
            else
                q4_store<float>(static_cast<float*>(p.a.out) + o, p.a.res ? static_cast<const float*>(p.a.res) + o : nullptr,
                                y, p.a.bias, n);
        };
        if (wk == 1 && csize == 1 && !any_direct) {
#pragma unroll
            for (int o = 0; o < C::kOut; o++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (mine(o, i)) put(8 * o + mt + (i & 1), row + 8 * (i >> 1), v[o][i]);
            continue;
        }
        // ---- the tile's sums: warps in order, then cluster ranks in order
        float* rbuf = red + parity * warps * C::kSums;
        float* wsum = rbuf + warp * C::kSums;  // [token][row]
#pragma unroll
        for (int o = 0; o < C::kOut; o++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (mine(o, i)) wsum[(8 * o + mt + (i & 1)) * 16 + row + 8 * (i >> 1)] = v[o][i];
        if (any_direct && tile < p.tiles) {  // rare: infinities or NaN among this CTA's elements
            __syncwarp();
            for (int m = 0; m < M; m++)
                for (int c = kw; c < xchunks; c += wk)
                    if (direct[m * xchunks + c]) direct_chunk(p.a, wsum + m * 16, tile, m0 + m, ch0 * C::kChunks + c);
        }
        if (wk == 1)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(wk * 32) : "memory");
        const int gt = kw * 32 + lane, outs = M * 16;
        const float* gsum = rbuf + group * wk * C::kSums;
        auto warp_sums = [&](int e) {
            float y = gsum[e];
#pragma unroll 4
            for (int w = 1; w < wk; w++) y += gsum[w * C::kSums + e];
            return y;
        };
        if (csize == 1) {
            for (int e = gt; e < outs; e += wk * 32) put(e >> 4, e & 15, warp_sums(e));
        } else {
            // Rank 0 collects.  The others go on and wait for this tile's barrier before they store for the
            // next: by then rank 0 has read what their buffer held two tiles ago.
            if (it > 0 && rank != 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            float* to = cluster.map_shared_rank(cbuf, 0) + ((parity * csize + rank) * groups + group) * C::kSums;
            for (int e = gt; e < outs; e += wk * 32) to[e] = warp_sums(e);
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            if (rank == 0) {
                asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
                const float* from = cbuf + (parity * csize * groups + group) * C::kSums;
                for (int e = gt; e < outs; e += wk * 32) {
                    float y = from[e];
                    for (int c = 1; c < csize; c++) y += from[c * groups * C::kSums + e];
                    put(e >> 4, e & 15, y);
                }
                __syncwarp();
            }
        }
        if (wk == 1 && csize == 1)
            __syncwarp();  // the one buffer is read
        else
            parity ^= 1;
    }
    if (!ok && lane == 0)  // copies still in flight land before the CTA ends
        for (int i = 0; i < inflight; i++) {
            tc::mbar_wait(bar0 + 8 * stage, phase, &zero, kWaitNs);
            if (++stage == p.stages) stage = 0, phase ^= 1;
        }
    if (csize > 1) {
        if (rounds > 0 && rank != 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        cluster.sync();  // rank 0's memory outlives the stores into it
    }
}

constexpr size_t kSmemPerSM = 228 * 1024;

struct StreamPlan {
    int tokens = 0;  // of one launch; 0: the kernel cannot take the shape
    bool halves = false;
    int nt = 0, ib = 1, cluster = 1, nch = 0, per = 0, warps = 8, wk = 8, stages = 0;
};

template <int NT, int G, int IB, bool kHalves>
cudaError_t launch_stream(const StreamParams& p, const StreamPlan& s, int num_sms, size_t max_smem, cudaStream_t stream)
{
    using C = StreamCfg<NT, IB, kHalves>;
    CUtensorMap mw;
    TmapDesc w{};
    w.base = p.a.q4;
    w.inner = p.a.K / 2;
    w.outer = p.a.N;
    w.row_bytes = p.a.K / 2;
    w.box_inner = 128;
    w.box_outer = 16;
    w.dtype = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    w.swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
    if (!tmap_2d(&mw, w)) return cudaErrorInvalidValue;
    auto kern = q4_stream_kernel<NT, G, IB, kHalves>;
    static thread_local bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)max_smem);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int groups = s.warps / p.wk;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((unsigned)s.warps * 32);
    cfg.dynamicSmemBytes = C::smem(s.warps, p.stages, p.tokens, p.per, s.cluster, p.wk);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)s.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.cluster > 1 ? 2 : 1;
    // As many CTAs (clusters) as the device holds at a time.  The hardware's own count: a cluster stays
    // within a GPC, so fewer fit than the SMs would hold.
    int resident = (s.warps == 8 && 2 * cfg.dynamicSmemBytes + 2048 <= kSmemPerSM ? 2 : 1) * num_sms;
    if (s.cluster > 1) {
        struct Known {
            int dev, cluster, warps, n;
            size_t smem;
        };
        static thread_local Known known[16];
        static thread_local int used = 0, next = 0;
        int i = 0;
        while (i < used && !(known[i].dev == dev && known[i].cluster == s.cluster && known[i].warps == s.warps &&
                             known[i].smem == cfg.dynamicSmemBytes))
            i++;
        if (i == used) {
            Known k{dev, s.cluster, s.warps, 0, cfg.dynamicSmemBytes};
            cfg.gridDim = dim3((unsigned)s.cluster);
            cfg.attrs = attr + 1;
            cfg.numAttrs = 1;
            if ((e = cudaOccupancyMaxActiveClusters(&k.n, kern, &cfg)) != cudaSuccess) return e;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            i = used < 16 ? used++ : next++ % 16;
            known[i] = k;
        }
        resident = std::max(1, known[i].n);
    }
    // Of several passes over the weights those that fit run side by side, and a CTA puts its tokens into shared
    // memory once for all its tiles: as many per pass as end soonest (the tokens count as two rounds of tiles).
    const int passes = (p.M + p.tokens - 1) / p.tokens, turns = (p.tiles + groups - 1) / groups;
    int wide = std::min(turns, resident);
    if (passes > 1) {
        double best = 1e30;
        for (int g = wide; g >= 1; g--) {
            const double cost = (double)(((long long)g * passes + resident - 1) / resident) * ((turns + g - 1) / g + 2);
            if (cost < best) best = cost, wide = g;
        }
    }
    cfg.gridDim = dim3((unsigned)(wide * s.cluster), (unsigned)passes);
    e = cudaLaunchKernelEx(&cfg, kern, mw, p);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <int NT, int G, bool kHalves>
cudaError_t launch_stream_ib(const StreamParams& p, const StreamPlan& s, int num_sms, size_t max_smem, cudaStream_t stream)
{
    return s.ib == 1 ? launch_stream<NT, G, 1, kHalves>(p, s, num_sms, max_smem, stream)
                     : launch_stream<NT, G, 2, kHalves>(p, s, num_sms, max_smem, stream);
}

template <int G>
cudaError_t launch_stream_nt(const StreamParams& p, const StreamPlan& s, int num_sms, size_t max_smem, cudaStream_t stream)
{
    if (s.halves)
        return s.nt == 1 ? launch_stream_ib<1, G, true>(p, s, num_sms, max_smem, stream)
                         : launch_stream_ib<2, G, true>(p, s, num_sms, max_smem, stream);
    return s.nt == 1 ? launch_stream_ib<1, G, false>(p, s, num_sms, max_smem, stream)
                     : launch_stream_ib<3, G, false>(p, s, num_sms, max_smem, stream);
}

size_t stream_smem(int nt, int ib, bool halves, int warps, int stages, int M, int per, int cluster, int wk)
{
    auto of = [&](auto one, auto two) {
        return ib == 1 ? decltype(one)::smem(warps, stages, M, per, cluster, wk) : decltype(two)::smem(warps, stages, M, per, cluster, wk);
    };
    if (halves)
        return nt == 1 ? of(StreamCfg<1, 1, true>(), StreamCfg<1, 2, true>())
                       : of(StreamCfg<2, 1, true>(), StreamCfg<2, 2, true>());
    return nt == 1 ? of(StreamCfg<1, 1, false>(), StreamCfg<1, 2, false>())
                   : of(StreamCfg<3, 1, false>(), StreamCfg<3, 2, false>());
}

constexpr int kMaxCluster = 8;

// Items of two boxes where a row has several (a wait, a copy and their bookkeeping cost about as much as a
// box's products: 37888 x 3584, one token, 14.9 us with one box, 13.4 with two), two items in flight a warp
// (three: 14.4 us, the copies' queue then holds up the warps); sixteen warps an SM, in two CTAs where the
// tokens leave room, else in one, else in clusters of 2, 4, 8; eight only where that does not fit either
// (8 tokens in bytes, 4096 x 14336: 17 us in clusters of four, with eight warps in clusters of two 26).
// One or two tokens take a cluster only where one CTA cannot hold them.  With more, putting them into shared memory
// is what a CTA of few tiles spends its time on, so a long K is split over as many SMs as the tiles
// leave free (8 tokens in bytes, 896 x 4864: 9.6 us on clusters of two, 12 without), and over more where
// that leaves warps less to do (9 tokens, 14336 x 8192: 32 us in clusters of two, in single CTAs 48).
StreamPlan plan_stream(const Q4Args& a, size_t M, long long passes, int num_sms, size_t max_smem)
{
    const long long tiles = (long long)((a.N + 15) / 16) * passes;
    const bool f16 = a.in_dtype == kF16;
    for (int m = (int)std::min<size_t>(M, f16 ? kMaxTokens : kMaxDigitTokens); m >= 1; m--) {
        const bool halves = f16 && m > 2;
        const int nt = m <= 2 ? 1 : !halves ? 3 : m <= 8 ? 1 : 2;
        int c0 = 1;
        while (m > 2 && c0 < kMaxCluster && 2 * c0 * tiles <= num_sms && a.K >= (size_t)4096 * c0) c0 *= 2;
        for (int all = 1; all >= 0; all--) {
            StreamPlan found;
            double best = 1e30;  // what a warp has to do, in boxes
            for (int c = all ? c0 : 1; c <= kMaxCluster && !(m <= 2 && found.tokens); c *= 2)
                for (int ib = all && a.K >= 2048 && (m <= 2 || c == 1) ? 2 : 1; ib >= 1; ib--) {
                    StreamPlan s;
                    s.tokens = m;
                    s.halves = halves;
                    s.nt = nt;
                    s.ib = ib;
                    s.cluster = c;
                    s.nch = (int)((a.K + ib * kBoxK - 1) / (ib * kBoxK));
                    s.per = (s.nch + c - 1) / c;
                    if ((s.nch + s.per - 1) / s.per != c) continue;  // a rank would have nothing
                    // Warps that share a tile (two at least in a cluster, whose rank 0 holds every group's sums): those that
                    // end soonest, an item costing a third of a box beside its boxes, and the joining of their sums.
                    auto fit = [&](int warps, size_t budget) {
                        const long long slots = c == 1 ? num_sms * 16 : num_sms / c * warps;
                        bool any = false;
                        s.warps = warps;
                        for (s.wk = c > 1 ? 2 : 1; s.wk <= warps; s.wk *= 2) {
                            s.stages = ib == 2 ? 2 : 3;
                            while (s.stages >= 2 && stream_smem(nt, ib, halves, warps, s.stages, m, s.per, c, s.wk) > budget) s.stages--;
                            if (s.stages < 2) continue;
                            any = true;
                            const double join = c > 1 ? 2.7 : s.wk > 1 ? 1.5 : 0.75;
                            const double cost = (double)((tiles * s.wk + slots - 1) / slots) * ((s.per + s.wk - 1) / s.wk * (ib + 0.33) + join) * (c > c0 ? 1.15 : 1.0);
                            if (cost < best) best = cost, found = s;
                        }
                        return any;
                    };
                    if (!all)
                        fit(8, max_smem);
                    else if (c > 1 || !fit(8, kSmemPerSM / 2 - 1024))
                        fit(16, max_smem);
                }
            if (found.tokens) return found;
        }
    }
    return StreamPlan{};
}

}  // namespace

bool q4_stream_supports(const Q4Args& a)
{
    return a.K % 32 == 0 && (uintptr_t)a.q4 % 16 == 0 && (uintptr_t)a.x % 16 == 0 &&
           a.N <= (size_t)INT32_MAX - 4096 && encode_fn() != nullptr;
}

cudaError_t launch_q4_stream(const Q4Args& a, int num_sms, size_t max_smem, cudaStream_t stream)
{
    if (!q4_stream_supports(a)) return cudaErrorNotSupported;
    const size_t ib = a.in_dtype == kF16 ? 2 : 4, ob = a.out_dtype == kF16 ? 2 : 4;
    const StreamPlan most = plan_stream(a, a.M, 1, num_sms, max_smem);
    if (!most.tokens) return cudaErrorNotSupported;  // one token's slice exceeds the shared memory
    // Passes of as good as equal numbers of tokens, up to 32768 of them to a launch.
    const size_t passes = (a.M + most.tokens - 1) / most.tokens, tokens = (a.M + passes - 1) / passes;
    const StreamPlan s = passes == 1 ? most : plan_stream(a, tokens, (long long)passes, num_sms, max_smem);
    for (size_t m0 = 0; m0 < a.M;) {
        StreamParams p;
        p.a = a;
        p.a.x = static_cast<const char*>(a.x) + m0 * a.K * ib;
        p.a.out = static_cast<char*>(a.out) + m0 * a.N * ob;
        p.a.res = a.res ? static_cast<const char*>(a.res) + m0 * a.N * ob : nullptr;
        p.tokens = s.tokens;
        p.M = (int)std::min(a.M - m0, (size_t)s.tokens * 32768);
        p.wk = s.wk;
        p.wk_log2 = s.wk == 16 ? 4 : s.wk == 8 ? 3 : s.wk == 4 ? 2 : s.wk == 2 ? 1 : 0;
        p.stages = s.stages;
        p.nch = s.nch;
        p.per = s.per;
        p.tiles = (int)((a.N + 15) / 16);
        cudaError_t e = a.group == 32   ? launch_stream_nt<32>(p, s, num_sms, max_smem, stream)
                        : a.group == 64 ? launch_stream_nt<64>(p, s, num_sms, max_smem, stream)
                                        : launch_stream_nt<128>(p, s, num_sms, max_smem, stream);
        if (e != cudaSuccess) return e;
        m0 += (size_t)p.M;
    }
    return cudaSuccess;
}

cudaError_t read_kernel_error_q4(int* code, bool clear)
{
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_q4_error, sizeof(int));
    if (e != cudaSuccess) return e;
    *code = v;
    if (clear && v) {
        const int z = 0;
        e = cudaMemcpyToSymbol(g_q4_error, &z, sizeof(int));
    }
    return e;
}

cudaError_t launch_q4_linear_generic(const Q4Args& a, cudaStream_t stream)
{
    if (a.in_dtype == kF16)
        return a.out_dtype == kF16 ? launch_generic<__half, __half>(a, stream) : launch_generic<__half, float>(a, stream);
    return a.out_dtype == kF16 ? launch_generic<float, __half>(a, stream) : launch_generic<float, float>(a, stream);
}

}  // namespace b200q8
