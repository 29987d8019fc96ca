// logits.cu -- from a step's logits to its token: penalties for tokens already there, biases, an
// allowed-token mask and the greedy choice, in one pass over the logits.
//
// Per row m and token i, in fp32 (each line rounded once, as written):
//   v = logits[m, i]
//   i in the row's history:              v = v > 0 ? v / repetition : v * repetition
//   i c > 0 times behind the prompt:     v = v - frequency * c;  v = v - presence
//   i in the row's bias list:            v = v + bias            (a token listed twice: its last entry)
//   i not allowed:                       v = -inf                (whatever v was, NaN included)
//   out[m, i] = v in the output type; argmax[m] = first largest of the allowed, as stored.
//
// A cluster of eight CTAs serves one row: each CTA owns a slice of the vocabulary, counts the history's
// tokens of its slice in shared memory (integer atomics, so the order does not matter), then passes
// over its logits once, four tokens a thread and step.  The CTAs' best tokens meet in the first CTA's
// shared memory.  No workspace, so calls may overlap in any way.
//
// Bound by HBM (the logits read and written once) for batches, by launch and latency for a few rows.
// Counts take 16 bits where the history cannot exceed them, so that four CTAs of 256 threads fit an SM at a
// vocabulary of 152064; a few rows take 1024 threads a CTA instead, as more SMs than CTAs are there.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace b200q8 {

namespace {

constexpr int kMaxThreads = 1024;
constexpr int kLogitCluster = 8;

// Unsigned key of a float that is no NaN: larger value, larger key; -0 and +0 alike.
__device__ __forceinline__ uint32_t order_key(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The greedy choice in std::max_element's order over the allowed tokens: the first stays unless a later
// one is larger.  So a NaN wins only as the first; where nothing exceeds -inf the first allowed wins;
// else the first of the largest.
struct Choice {
    float top = -INFINITY;
    uint32_t at = 0;       // the first token of value `top`, if top > -inf
    uint32_t first = ~0u;  // the first allowed token
    bool first_nan = false;
};

// Per-token state in shared memory: a count (the token's occurrences behind the prompt, and in the top
// bit whether it is in the prompt) and the last bias entry + 1, of 16 or 32 bits each.  Slot u of the words s.
template <bool kWide>
struct Slots;
template <>
struct Slots<true> {
    static constexpr int kBytes = 4;
    static constexpr uint32_t kInPrompt = 0x80000000u;
    static __device__ __forceinline__ void add(uint32_t* s, int u) { atomicAdd(s + u, 1u); }
    static __device__ __forceinline__ void mark(uint32_t* s, int u) { atomicOr(s + u, kInPrompt); }
    static __device__ __forceinline__ void raise(uint32_t* s, int u, uint32_t v) { atomicMax(s + u, v); }
    static __device__ __forceinline__ uint32_t load(const uint32_t* s, int u) { return s[u]; }
    static __device__ __forceinline__ void load4(const uint32_t* s, int u, uint32_t (&c)[4])
    {
        const uint4 v = *reinterpret_cast<const uint4*>(s + u);
        c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
    }
};
template <>
struct Slots<false> {
    static constexpr int kBytes = 2;
    static constexpr uint32_t kInPrompt = 0x8000u;
    static __device__ __forceinline__ void add(uint32_t* s, int u) { atomicAdd(s + (u >> 1), 1u << (16 * (u & 1))); }  // at most 32767
    static __device__ __forceinline__ void mark(uint32_t* s, int u) { atomicOr(s + (u >> 1), kInPrompt << (16 * (u & 1))); }
    static __device__ __forceinline__ void raise(uint32_t* s, int u, uint32_t v)
    {
        const int sh = 16 * (u & 1);
        uint32_t old = s[u >> 1];
        while (((old >> sh) & 0xFFFFu) < v) {  // ends: a failed exchange is another's success, and each raises a value
            const uint32_t seen = atomicCAS(s + (u >> 1), old, (old & ~(0xFFFFu << sh)) | (v << sh));
            if (seen == old) break;
            old = seen;
        }
    }
    static __device__ __forceinline__ uint32_t load(const uint32_t* s, int u) { return (s[u >> 1] >> (16 * (u & 1))) & 0xFFFFu; }
    static __device__ __forceinline__ void load4(const uint32_t* s, int u, uint32_t (&c)[4])
    {
        const uint2 v = *reinterpret_cast<const uint2*>(s + (u >> 1));
        c[0] = v.x & 0xFFFFu, c[1] = v.x >> 16, c[2] = v.y & 0xFFFFu, c[3] = v.y >> 16;
    }
};

__device__ __forceinline__ void load4(const float* p, float (&v)[4])
{
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&v)[4])
{
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
    v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4])
{
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__half* p, const float (&v)[4])
{
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <typename OT>
__device__ __forceinline__ float as_stored(float v)
{
    if constexpr (sizeof(OT) == 2)
        return __half2float(__float2half_rn(v));
    else
        return v;
}

template <typename IT, typename OT, bool kWide>
__global__ void __launch_bounds__(kMaxThreads) logits_kernel(const LogitArgs a, int slice)
{
    using S = Slots<kWide>;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long m = blockIdx.x / C;
    const int tid = threadIdx.x, nt = blockDim.x;
    extern __shared__ __align__(16) uint32_t slots[];
    __shared__ unsigned long long red[2][kMaxThreads / 32], joined[2][16];

    const int V = (int)a.V;
    const IT* in = static_cast<const IT*>(a.logits) + m * (long long)a.in_stride;
    OT* out = a.out ? static_cast<OT*>(a.out) + m * (long long)a.out_stride : nullptr;
    // Four tokens at a time from the first whose logit is aligned to four elements; where the outputs are
    // not aligned with them, one at a time.
    const int lead = (int)((4 - (reinterpret_cast<uintptr_t>(in) / sizeof(IT) & 3)) & 3);  // of the row, so of any slice
    const bool vec = !out || ((reinterpret_cast<uintptr_t>(out) / sizeof(OT) + lead) & 3) == 0;
    pdl_wait();
    pdl_launch_dependents();
    if (tid == 0) {  // the first slice's logits into L2 while the lists are read
        const long long b0 = (long long)rank * slice, n0 = min((long long)slice, V - b0);
        const uintptr_t p0 = (reinterpret_cast<uintptr_t>(in + b0) + 15) & ~(uintptr_t)15;
        const long long bytes = n0 > 0 ? (long long)(reinterpret_cast<uintptr_t>(in + b0 + n0) - p0) & ~15LL : 0;
        if (bytes > 0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p0), "r"((uint32_t)bytes) : "memory");
    }
    const int* hist = a.history ? a.history + m * (long long)a.history_stride : nullptr;
    const int hlen = hist ? max(0, min(a.history_len[m], (int)a.history_count)) : 0;
    const int plen = hist && a.prompt_len ? max(0, min(a.prompt_len[m], hlen)) : 0;
    const int* bids = a.bias_ids ? a.bias_ids + m * (long long)a.bias_stride : nullptr;
    const int blen = !bids ? 0 : a.bias_len ? max(0, min(a.bias_len[m], (int)a.bias_count)) : (int)a.bias_count;
    const float* bval = bids ? a.bias_values + m * (long long)a.bias_stride : nullptr;
    const float rep = a.repetition ? a.repetition[m] : 1.0f;
    const float pres = a.presence ? a.presence[m] : 0.0f;
    const float freq = a.frequency ? a.frequency[m] : 0.0f;
    const uint32_t* mask = a.allowed ? a.allowed + m * (long long)a.allowed_stride : nullptr;
    // Slots of the slice's tokens, placed so that those of an aligned four are aligned too.
    const int room = slice + 8;
    const int count = (4 - lead) & 3, entry = count + (a.history ? room : 0);

    Choice best;
    // The rules on one token; what is stored, as a float.
    auto rules = [&](float v, int tok, uint32_t c, uint32_t e, bool ok) {
        if (c) {
            v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            const uint32_t made = c & ~S::kInPrompt;
            if (made) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)made)), pres);
        }
        if (e) v = __fadd_rn(v, bval[e - 1]);
        if (!ok) v = -INFINITY;
        v = as_stored<OT>(v);
        if (v > best.top) best.top = v, best.at = (uint32_t)tok;
        return v;
    };
    for (long long base = (long long)rank * slice; base < V; base += (long long)C * slice) {
        const int n = (int)min((long long)slice, V - base);
        {
            uint4* z = reinterpret_cast<uint4*>(slots);
            const int lists = blen && a.history ? 2 : hlen || blen ? 1 : 0;  // of a history alone the first
            const int clear = lists * room * S::kBytes / 16;
            for (int i = tid; i < clear; i += nt) z[i] = make_uint4(0, 0, 0, 0);
        }
        if (hlen || blen) __syncthreads();
#pragma unroll 8
        for (int j = tid; j < hlen; j += nt) {
            const long long u = (long long)hist[j] - base;
            if (u >= 0 && u < n) {
                if (j < plen)
                    S::mark(slots, count + (int)u);
                else
                    S::add(slots, count + (int)u);
            }
        }
        for (int j = tid; j < blen; j += nt) {
            const long long u = (long long)bids[j] - base;
            if (u >= 0 && u < n) S::raise(slots, entry + (int)u, (uint32_t)(j + 1));
        }
        if (hlen || blen) __syncthreads();

        auto one = [&](int i) {
            const int tok = (int)base + i;
            const bool ok = !mask || ((__ldg(mask + (tok >> 5)) >> (tok & 31)) & 1u);
            const float v = rules(load_as_f32<IT>(in + tok), tok, hlen ? S::load(slots, count + i) : 0u,
                                  blen ? S::load(slots, entry + i) : 0u, ok);
            if (out) store_from_f32<OT>(out + tok, v);
            if (ok && best.first == ~0u) best.first = (uint32_t)tok, best.first_nan = v != v;
        };
        if (vec) {
            const int head = min(lead, n), fours = (n - head) / 4, tail = head + 4 * fours;
            if (tid < head) one(tid);
            constexpr int U = 4;
            for (int q0 = tid; q0 < fours; q0 += U * nt) {
                float v[U][4];
                uint32_t w[U];
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int q = q0 + k * nt;
                    if (q < fours) {
                        const int tok = (int)base + head + 4 * q;
                        load4(in + tok, v[k]);
                        w[k] = ~0u;
                        if (mask) {
                            const uint32_t lo = __ldg(mask + (tok >> 5));
                            const uint32_t hi = (tok & 31) > 28 ? __ldg(mask + (tok >> 5) + 1) : 0u;  // a lead of 1 .. 3
                            w[k] = __funnelshift_r(lo, hi, tok & 31);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < U; k++) {
                    const int q = q0 + k * nt;
                    if (q >= fours) break;
                    const int i = head + 4 * q, tok = (int)base + i;
                    uint32_t c[4] = {}, e[4] = {};
                    if (hlen) S::load4(slots, count + i, c);
                    if (blen) S::load4(slots, entry + i, e);
#pragma unroll
                    for (int j = 0; j < 4; j++) v[k][j] = rules(v[k][j], tok + j, c[j], e[j], (w[k] >> j) & 1u);
                    if (out) store4(out + tok, v[k]);
                    if (best.first == ~0u && (w[k] & 15u)) {
                        const int j = __ffs(w[k] & 15u) - 1;
                        best.first = (uint32_t)(tok + j);
                        const float f = j == 0 ? v[k][0] : j == 1 ? v[k][1] : j == 2 ? v[k][2] : v[k][3];
                        best.first_nan = f != f;
                    }
                }
            }
            if (tid < n - tail) one(tail + tid);
        } else {
#pragma unroll 4
            for (int i = tid; i < n; i += nt) one(i);
        }
        if (base + (long long)C * slice < V && (hlen || blen)) __syncthreads();  // the next slice clears the slots
    }
    if (!a.argmax) return;
    // (value, complement of the token): the larger wins, then the lower token; (first token, NaN): the lower
    unsigned long long b = best.top > -INFINITY ? ((unsigned long long)order_key(best.top) << 32) | (uint32_t)~best.at : 0ull;
    unsigned long long f = best.first == ~0u ? ~0ull : ((unsigned long long)best.first << 1) | (best.first_nan ? 1u : 0u);
    auto join = [&](unsigned long long b2, unsigned long long f2) {
        b = b2 > b ? b2 : b;
        f = f2 < f ? f2 : f;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, b, o), __shfl_xor_sync(0xffffffffu, f, o));
    if ((tid & 31) == 0) {
        red[0][tid >> 5] = b;
        red[1][tid >> 5] = f;
    }
    __syncthreads();
    if (tid < 32) {
        b = tid < nt / 32 ? red[0][tid] : 0ull;
        f = tid < nt / 32 ? red[1][tid] : ~0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, b, o), __shfl_xor_sync(0xffffffffu, f, o));
    }
    cluster.sync();  // rank 0 runs (its memory may be stored to)
    if (tid == 0) {
        unsigned long long* to = cluster.map_shared_rank(&joined[0][0], 0);
        to[rank] = b;
        to[16 + rank] = f;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        b = 0ull;
        f = ~0ull;
        for (int r = 0; r < C; r++) join(joined[0][r], joined[1][r]);
        a.argmax[m] = f == ~0ull ? -1 : (f & 1) || b == 0ull ? (int)(f >> 1) : (int)~(uint32_t)b;
    }
}

template <typename IT, typename OT, bool kWide>
cudaError_t launch_sized(const LogitArgs& a, int num_sms, size_t max_smem, cudaStream_t stream)
{
    auto kern = logits_kernel<IT, OT, kWide>;
    constexpr size_t kBytes = Slots<kWide>::kBytes;
    const size_t lists = (a.history ? 1 : 0) + (a.bias_ids ? 1 : 0);
    const size_t budget = max_smem - 4096;  // beside the static part
    // A slice is whole mask words; its slots are 8 more than its tokens, and 4 behind the last list's.
    long long slice = ((long long)a.V + kLogitCluster - 1) / kLogitCluster;
    slice = (slice + 31) / 32 * 32;
    if (lists) slice = std::min<long long>(slice, (long long)(budget / (lists * kBytes) - 24) / 32 * 32);
    const size_t smem = lists ? (lists * (size_t)(slice + 8) + 8) * kBytes : 0;
    static thread_local bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)budget);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.M * kLogitCluster));
    cfg.blockDim = dim3(a.M * kLogitCluster <= (size_t)num_sms ? 1024 : 256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kLogitCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, a, (int)slice);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename IT, typename OT>
cudaError_t launch_typed(const LogitArgs& a, int num_sms, size_t max_smem, cudaStream_t stream)
{
    const bool wide = (a.history && a.history_count > 32767) || (a.bias_ids && a.bias_count > 65534);
    return wide ? launch_sized<IT, OT, true>(a, num_sms, max_smem, stream)
                : launch_sized<IT, OT, false>(a, num_sms, max_smem, stream);
}

}  // namespace

cudaError_t launch_logits(const LogitArgs& a, int num_sms, size_t max_smem, cudaStream_t stream)
{
    if (a.in_dtype == kF16)
        return a.out_dtype == kF16 ? launch_typed<__half, __half>(a, num_sms, max_smem, stream)
                                   : launch_typed<__half, float>(a, num_sms, max_smem, stream);
    return a.out_dtype == kF16 ? launch_typed<float, __half>(a, num_sms, max_smem, stream)
                               : launch_typed<float, float>(a, num_sms, max_smem, stream);
}

}  // namespace b200q8
