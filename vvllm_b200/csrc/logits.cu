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
// A cluster of four or eight CTAs serves one row.  Its tokens are dealt to them in blocks of 1024 (frequent
// tokens have neighbouring numbers: contiguous slices left one CTA with most of the work).  Each CTA
//   - counts the history's tokens of its blocks, and notes the last bias entry of each, in shared memory
//     (integer atomics, so the order does not matter), listing every token it meets once, and in a bitmap;
//   - passes over its logits once, four tokens a thread and step, and leaves the named ones as they are;
//   - works out the named tokens one by one, a thread each.
// (Penalties within the pass would cost their division wherever one of a warp's 128 tokens has been seen.)
// The CTAs' best tokens meet in the first CTA's shared memory.  No workspace, so calls may overlap in any way.
//
// Bound by HBM (the logits read and written once) for batches, by launch and latency for a few rows.
// Slots take 16 bits where the lists' lengths allow, so that two CTAs of 512 threads fit an SM at a
// vocabulary of 152064.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace b200q8 {

namespace {

constexpr int kThreads = 512;
constexpr size_t kStaticSmem = 4096;  // left to the kernel's static shared memory

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
    uint32_t at = ~0u;     // the first token of value `top`, if top > -inf
    uint32_t first = ~0u;  // the first allowed token
    bool first_nan = false;
    __device__ __forceinline__ void take(float v, uint32_t tok)  // in any order
    {
        if (v > top || (v == top && tok < at)) top = v, at = tok;
        if (tok < first) first = tok, first_nan = v != v;
    }
};

// The same as numbers that join in any order: the value's key (0: none above -inf) with its token, and the
// first allowed token * 2 + (it is NaN).
struct Keys {
    uint32_t key, at, first;
    __device__ __forceinline__ explicit Keys(const Choice& c)
        : key(c.top > -INFINITY ? order_key(c.top) : 0u), at(c.at), first(c.first == ~0u ? ~0u : c.first * 2 + (c.first_nan ? 1u : 0u))
    {
    }
    __device__ __forceinline__ void join(uint32_t k, uint32_t a, uint32_t f)
    {
        if (k > key || (k == key && a < at)) key = k, at = a;
        first = min(first, f);
    }
    __device__ __forceinline__ void join_warp()
    {
        const uint32_t k = __reduce_max_sync(0xffffffffu, key);
        at = __reduce_min_sync(0xffffffffu, key == k ? at : ~0u);
        key = k;
        first = __reduce_min_sync(0xffffffffu, first);
    }
    __device__ __forceinline__ int token() const
    {
        return first == ~0u ? -1 : (first & 1u) || key == 0u ? (int)(first >> 1) : (int)at;
    }
};

// Per-token state in shared memory: a count (the token's occurrences behind the prompt, and in the top
// bit whether it is in the prompt) and the last bias entry + 1, of 16 or 32 bits each.  Slot u of the words s.
// add and mark return whether the slot was untouched.
template <bool kWide>
struct Slots;
template <>
struct Slots<true> {
    using Listed = uint32_t;
    static constexpr int kBytes = 4;
    static constexpr uint32_t kInPrompt = 0x80000000u;
    static __device__ __forceinline__ bool add(uint32_t* s, int u) { return atomicAdd(s + u, 1u) == 0; }
    static __device__ __forceinline__ bool mark(uint32_t* s, int u) { return atomicOr(s + u, kInPrompt) == 0; }
    static __device__ __forceinline__ void raise(uint32_t* s, int u, uint32_t v) { atomicMax(s + u, v); }
    static __device__ __forceinline__ uint32_t load(const uint32_t* s, int u) { return s[u]; }
};
template <>
struct Slots<false> {
    using Listed = uint16_t;
    static constexpr int kBytes = 2;
    static constexpr uint32_t kInPrompt = 0x8000u;
    static __device__ __forceinline__ bool add(uint32_t* s, int u)  // at most 32767 times
    {
        const int sh = 16 * (u & 1);
        return ((atomicAdd(s + (u >> 1), 1u << sh) >> sh) & 0xFFFFu) == 0;
    }
    static __device__ __forceinline__ bool mark(uint32_t* s, int u)
    {
        const int sh = 16 * (u & 1);
        return ((atomicOr(s + (u >> 1), kInPrompt << sh) >> sh) & 0xFFFFu) == 0;
    }
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

constexpr int kBlock = 1024;  // tokens dealt at a time

// A CTA's view of its row.
template <typename IT, typename OT, int C>  // C: CTAs of a row
struct Row {
    const IT* in;
    OT* out;               // or null
    const uint32_t* mask;  // or null
    int V, lead, rank;
    // The bits of tok .. tok + n - 1 (n <= 4) that are allowed.
    __device__ __forceinline__ uint32_t allowed(int tok, int n) const
    {
        const uint32_t all = (1u << n) - 1u;
        if (!mask) return all;
        const uint32_t lo = __ldg(mask + (tok >> 5));
        const uint32_t hi = (tok & 31) + n > 32 ? __ldg(mask + (tok >> 5) + 1) : 0u;
        return __funnelshift_r(lo, hi, tok & 31) & all;
    }
    // First token of this CTA's block k.
    __device__ __forceinline__ int block_token(int k) const { return lead + (rank + k * C) * kBlock; }
    // Calls f(slot) for a token that is this CTA's and of its blocks k0 .. k0 + room - 1 (slots of a block follow
    // one another; those of rank 0's tokens before the first block come last).
    template <class F>
    __device__ __forceinline__ void with_slot(int id, int k0, int room, F f) const
    {
        const uint32_t u = (uint32_t)id - (uint32_t)lead;  // huge for a negative id and for those before the blocks
        if (u / kBlock % C == (uint32_t)rank && u < (uint32_t)(V - lead)) {
            const int k = (int)(u / (kBlock * C)) - k0;
            if (k >= 0 && k < room) f(k * kBlock + (int)(u % kBlock));
        } else if ((uint32_t)id < (uint32_t)lead && rank == 0 && k0 == 0) {
            f(room * kBlock + id);
        }
    }
    __device__ __forceinline__ int slot_token(int u, int k0, int room) const
    {
        return u >= room * kBlock ? u - room * kBlock : block_token(k0 + u / kBlock) + u % kBlock;
    }
};

// Four tokens from tok.  ok: the allowed ones' bits; named: those worked out later, left as they are.
// w: the candidates' values.
template <typename IT, typename OT, bool kMask, bool kNamed>
__device__ __forceinline__ void four(float (&v)[4], float (&w)[4], uint32_t named, uint32_t ok)
{
    const uint32_t keep = ok | named;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (kMask) v[j] = keep & (1u << j) ? v[j] : -INFINITY;
        if (sizeof(IT) > sizeof(OT)) v[j] = as_stored<OT>(v[j]);
        w[j] = kNamed && (named & (1u << j)) ? -INFINITY : v[j];
    }
}

// Which of four equals top first.
__device__ __forceinline__ int place(const float (&w)[4], float top) { return w[0] == top ? 0 : w[1] == top ? 1 : w[2] == top ? 2 : 3; }

__device__ __forceinline__ void note_first(Choice& best, const float (&w)[4], int tok, uint32_t cand)
{
    if (best.first == ~0u && cand) {
        const int j = __ffs(cand) - 1;
        const float f = j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3];
        best.first = (uint32_t)(tok + j);
        best.first_nan = f != f;
    }
}

// Up to four tokens from tok, one by one in memory.
template <typename IT, typename OT, int C>
__device__ __noinline__ Choice few_tokens(const Row<IT, OT, C> r, int tok, int n, uint32_t named, Choice best)
{
    float v[4], w[4];
    for (int j = 0; j < 4; j++) v[j] = j < n ? load_as_f32<IT>(r.in + tok + j) : 0.0f;
    const uint32_t ok = r.allowed(tok, n);
    four<IT, OT, true, true>(v, w, named, ok);
    for (int j = 0; j < 4; j++) {
        if (r.out && j < n) store_from_f32<OT>(r.out + tok + j, v[j]);
        if (w[j] > best.top) best.top = w[j], best.at = (uint32_t)(tok + j);
    }
    note_first(best, w, tok, ok & ~named);
    return best;
}

// This thread's fours of `blocks` blocks from k0, all tokens of which exist, with vector loads and stores.
template <typename IT, typename OT, int C, bool kMask, bool kNamed, bool kOut>
__device__ __forceinline__ void pass(const Row<IT, OT, C>& r, const uint32_t* bits, int k0, int blocks, Choice& best)
{
    constexpr int U = 4, kPer = kThreads / (kBlock / 4);  // blocks of a step
    constexpr int kStep = kPer * C * kBlock;              // tokens from one four of a thread to its next
    const int g = threadIdx.x & (kBlock / 4 - 1), kq = threadIdx.x / (kBlock / 4);
    int left = (blocks - kq + kPer - 1) / kPer, tok = r.block_token(k0 + kq) + 4 * g;
    const int msh = tok & 31, bsh = 4 * (g & 7);
    const IT* src = r.in + tok;
    OT* dst = r.out + (kOut ? tok : 0);
    const uint32_t* mw = r.mask + (kMask ? tok >> 5 : 0);
    bits += kq * (kBlock / 32) + (g >> 3);
    float top = best.top;
    int at = -1;  // the four that holds it
    auto step = [&](auto count) {
        constexpr int N = decltype(count)::value;
        float v[N][4];
        uint32_t ok[N], named[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            load4(src + i * kStep, v[i]);
            ok[i] = 15u;
            if (kMask) {
                ok[i] = __ldg(mw + i * (kStep / 32)) >> msh;
                if (msh > 28) ok[i] |= __ldg(mw + i * (kStep / 32) + 1) << (32 - msh);  // with a lead
            }
            named[i] = kNamed ? bits[i * kPer * (kBlock / 32)] >> bsh : 0u;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            float w[4];
            four<IT, OT, kMask, kNamed>(v[i], w, named[i] & 15u, ok[i] & 15u);
            const float m = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));  // skips NaN
            if (m > top) top = m, at = tok + i * kStep;
            if (best.first == ~0u) note_first(best, w, tok + i * kStep, ok[i] & ~named[i] & 15u);
            if (kOut) store4(dst + i * kStep, v[i]);
        }
        tok += N * kStep;
        src += N * kStep;
        dst += kOut ? N * kStep : 0;
        mw += N * (kStep / 32);
        bits += N * kPer * (kBlock / 32);
    };
    const uint32_t* bits0 = bits;
    const int tok0 = tok;
    for (; left >= U; left -= U) step(std::integral_constant<int, U>());
    for (; left > 0; left--) step(std::integral_constant<int, 1>());
    if (at < 0) return;
    // Which of the four it was: they hold now, read again, what they held (or, in place, what was stored).
    float v[4], w[4];
    load4(r.in + at, v);
    const uint32_t named = kNamed ? (bits0[(at - tok0) / kStep * kPer * (kBlock / 32)] >> bsh) & 15u : 0u;
    four<IT, OT, kMask, kNamed>(v, w, named, r.allowed(at, 4));
    best.top = top;
    best.at = (uint32_t)(at + place(w, top));
}

// The lists' tokens of the CTA's blocks k0 .. k0 + room - 1: counts, last bias entries, `bits` and `list`.
// While the first of them are on their way, `mine` blocks of logits are requested into L2 (before, they would
// keep the lists waiting).
template <typename IT, typename OT, int C, bool kWide>
__device__ __noinline__ void read_lists(const Row<IT, OT, C> r, int mine, const int* hist, int hlen, int plen, const int* bids, int blen,
                                        int k0, int room, uint32_t* bits, uint32_t* count, uint32_t* entry,
                                        typename Slots<kWide>::Listed* list, int* listed)
{
    using S = Slots<kWide>;
    const int tid = threadIdx.x;
    auto request = [&]() {
        for (int k = tid; k < mine; k += kThreads) {
            const int t0 = r.block_token(k), n = min(kBlock, r.V - t0);
            const uintptr_t p0 = (reinterpret_cast<uintptr_t>(r.in + t0) + 15) & ~(uintptr_t)15;
            const long long bytes = (long long)(reinterpret_cast<uintptr_t>(r.in + t0 + n) - p0) & ~15LL;
            if (bytes > 0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p0), "r"((uint32_t)bytes) : "memory");
        }
    };
    auto name = [&](int u) {
        list[atomicAdd(listed, 1)] = (typename S::Listed)u;
        atomicOr(bits + (u >> 5), 1u << (u & 31));
    };
    // Eight ids on their way where the history is long; two where it is short, since fetching the code of
    // eight takes longer than their loads do (200 ids: 6.5 us, with eight 6.7; 4096 ids in 64 rows: 27 us, with four 29).
    auto count_ids = [&](auto width) {
        constexpr int U = decltype(width)::value;
#pragma unroll 1
        for (int j0 = tid; j0 < hlen; j0 += U * kThreads) {
            int id[U];
#pragma unroll
            for (int i = 0; i < U; i++) id[i] = j0 + i * kThreads < hlen ? __ldg(hist + j0 + i * kThreads) : -1;
            if (j0 == tid && k0 == 0) request();
#pragma unroll
            for (int i = 0; i < U; i++)
                r.with_slot(id[i], k0, room, [&](int u) {
                    if (j0 + i * kThreads < plen ? S::mark(count, u) : S::add(count, u)) name(u);
                });
        }
    };
    if (hlen <= 2 * kThreads)
        count_ids(std::integral_constant<int, 2>());
    else
        count_ids(std::integral_constant<int, 8>());
    if (blen) {
        for (int j = tid; j < blen; j += kThreads)
            r.with_slot(__ldg(bids + j), k0, room, [&](int u) { S::raise(entry, u, (uint32_t)(j + 1)); });
        __syncthreads();
        for (int j = tid; j < blen; j += kThreads)  // a token is named by its last entry, if the history has not named it
            r.with_slot(__ldg(bids + j), k0, room, [&](int u) {
                if (S::load(entry, u) == (uint32_t)(j + 1) && !(hlen && S::load(count, u))) name(u);
            });
    }
}

template <typename IT, typename OT, bool kWide, int C>
__global__ void __launch_bounds__(kThreads, 2) logits_kernel(const LogitArgs a, int room)
{
    using S = Slots<kWide>;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    const int tid = threadIdx.x;
    extern __shared__ __align__(16) uint32_t slots[];
    __shared__ uint32_t red[3][kThreads / 32], joined[3][C];
    __shared__ int listed;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs

    Row<IT, OT, C> r;
    r.rank = rank;
    const long long m = blockIdx.x / C;
    r.V = (int)a.V;
    r.in = static_cast<const IT*>(a.logits) + m * (long long)a.in_stride;
    r.out = a.out ? static_cast<OT*>(a.out) + m * (long long)a.out_stride : nullptr;
    r.mask = a.allowed ? a.allowed + m * (long long)a.allowed_stride : nullptr;
    // Blocks start at the first token whose logit is aligned to four elements; rank 0 takes the up to three
    // before.  Where the outputs are not aligned with the logits, four are loaded and stored one by one.
    r.lead = min((int)((4 - (reinterpret_cast<uintptr_t>(r.in) / sizeof(IT) & 3)) & 3), r.V);
    const bool vec = !r.out || ((reinterpret_cast<uintptr_t>(r.out) / sizeof(OT) + r.lead) & 3) == 0;
    const int whole = (r.V - r.lead) / kBlock, blocks = (r.V - r.lead + kBlock - 1) / kBlock;  // of the row
    const int mine = (blocks - rank + C - 1) / C;  // of this CTA: block b is rank b % C's, its b / C th
    const int mine_whole = (whole - rank + C - 1) / C;
    pdl_wait();
    pdl_launch_dependents();
    const int hlen = a.history ? max(0, min(a.history_len[m], (int)a.history_count)) : 0;
    const int blen = !a.bias_ids ? 0 : a.bias_len ? max(0, min(a.bias_len[m], (int)a.bias_count)) : (int)a.bias_count;
    const bool lists = hlen > 0 || blen > 0;
    // Shared memory: a bit per token of `room` blocks at a time, and of rank 0's up to three tokens before
    // the first block (last); the counts' slots; the bias entries' slots; the named tokens' slot numbers.
    const int tokens = room * kBlock, bit_words = tokens / 32 + 4, slot_words = (tokens + 8) * S::kBytes / 4;
    uint32_t* bits = slots;
    uint32_t* count = bits + bit_words;
    uint32_t* entry = count + (a.history ? slot_words : 0);
    typename S::Listed* list = reinterpret_cast<typename S::Listed*>(entry + (a.bias_ids ? slot_words : 0));

    Choice best, best_named;
    for (int k0 = 0; k0 == 0 || k0 < mine; k0 += room) {
        if (lists) {
            if (k0) __syncthreads();  // the slots of the blocks before are read
            const int words = bit_words + (a.history ? slot_words : 0) + (blen ? slot_words : 0);
            for (int i = tid; i < words / 4; i += kThreads) reinterpret_cast<uint4*>(slots)[i] = make_uint4(0, 0, 0, 0);
            if (tid == 0) listed = 0;
            __syncthreads();
            const int plen = hlen && a.prompt_len ? max(0, min(a.prompt_len[m], hlen)) : 0;
            read_lists<IT, OT, C, kWide>(r, mine, a.history + m * (long long)a.history_stride, hlen, plen,
                                      a.bias_ids + m * (long long)a.bias_stride, blen, k0, room, bits, count, entry, list,
                                      &listed);
            __syncthreads();
        }
        const int n = vec ? min(room, mine_whole - k0) : 0;  // blocks passed over with vectors
        auto go = [&](auto masked, auto named) {
            constexpr bool kMask = decltype(masked)::value, kNamed = decltype(named)::value;
            if (r.out)
                pass<IT, OT, C, kMask, kNamed, true>(r, bits, k0, n, best);
            else
                pass<IT, OT, C, kMask, kNamed, false>(r, bits, k0, n, best);
        };
        if (r.mask)
            lists ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
        else
            lists ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
        // What is left: the row's last block if it is not whole (all blocks where outputs are not aligned), and the lead.
        for (int q = max(n, 0) * (kBlock / 4) + tid; q < min(room, mine - k0) * (kBlock / 4); q += kThreads) {
            const int tok = r.block_token(k0 + q / (kBlock / 4)) + q % (kBlock / 4) * 4;
            if (tok < r.V)
                best = few_tokens<IT, OT, C>(r, tok, min(4, r.V - tok), lists ? (bits[q >> 3] >> (4 * (q & 7))) & 15u : 0u, best);
        }
        if (k0 == 0 && rank == 0 && tid == 0 && r.lead) {
            // its own choice: these tokens come before those above
            const Choice c = few_tokens<IT, OT, C>(r, 0, r.lead, lists ? bits[tokens >> 5] & 15u : 0u, Choice());
            if (c.top >= best.top) best.top = c.top, best.at = c.at;
            if (c.first != ~0u) best.first = c.first, best.first_nan = c.first_nan;
        }
        if (lists) {
            __syncthreads();  // the named tokens' outputs hold their logits now
            const float rep = a.repetition ? a.repetition[m] : 1.0f;
            const float pres = a.presence ? a.presence[m] : 0.0f;
            const float freq = a.frequency ? a.frequency[m] : 0.0f;
            const float* bval = a.bias_values + m * (long long)a.bias_stride;
            for (int i = tid; i < listed; i += kThreads) {
                const int u = list[i], tok = r.slot_token(u, k0, room);
                const uint32_t c = hlen ? S::load(count, u) : 0u, made = c & ~S::kInPrompt;
                const uint32_t e = blen ? S::load(entry, u) : 0u;
                float v = load_as_f32<IT>(r.in + tok);
                if (c) v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                if (made) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)made)), pres);
                if (e) v = __fadd_rn(v, bval[e - 1]);
                const bool ok = r.allowed(tok, 1);
                v = as_stored<OT>(ok ? v : -INFINITY);
                if (r.out) store_from_f32<OT>(r.out + tok, v);
                if (ok) best_named.take(v, (uint32_t)tok);
            }
        }
    }
    if (!a.argmax) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    Keys keys(best);
    const Keys named_keys(best_named);
    keys.join(named_keys.key, named_keys.at, named_keys.first);
    __syncwarp();
    keys.join_warp();
    if ((tid & 31) == 0) {
        red[0][tid >> 5] = keys.key;
        red[1][tid >> 5] = keys.at;
        red[2][tid >> 5] = keys.first;
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // rank 0 runs: its memory may be stored to
    if (tid < 32) {
        const bool in_cta = tid < kThreads / 32;
        keys.key = in_cta ? red[0][tid] : 0u;
        keys.at = in_cta ? red[1][tid] : ~0u;
        keys.first = in_cta ? red[2][tid] : ~0u;
        keys.join_warp();
        if (tid == 0) {
            uint32_t* to = cluster.map_shared_rank(&joined[0][0], 0);
            to[rank] = keys.key;
            to[C + rank] = keys.at;
            to[2 * C + rank] = keys.first;
        }
        __syncwarp();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0) {
        for (int q = 1; q < C; q++) keys.join(joined[0][q], joined[1][q], joined[2][q]);
        a.argmax[m] = keys.token();
    }
}

struct Plan {
    int room;     // blocks of a CTA that its slots hold at a time
    size_t smem;  // dynamic shared memory
};

template <bool kWide, int C>
Plan plan(const LogitArgs& a, size_t max_smem)
{
    constexpr size_t kBytes = Slots<kWide>::kBytes;
    using Listed = typename Slots<kWide>::Listed;
    const size_t lists = (a.history ? 1 : 0) + (a.bias_ids ? 1 : 0);
    long long room = (((long long)a.V + kBlock - 1) / kBlock + C - 1) / C;
    size_t smem = 0;
    if (lists) {
        if (!kWide) room = std::min<long long>(room, 63);  // slot numbers of 16 bits
        const size_t most = (a.history ? a.history_count : 0) + (a.bias_ids ? a.bias_count : 0);
        for (;; room--) {  // one block always fits
            const size_t tokens = (size_t)room * kBlock;
            smem = (tokens / 32 + 4) * 4 + lists * (tokens + 8) * kBytes + std::min(most, tokens + 4) * sizeof(Listed);
            if (smem <= max_smem - kStaticSmem) break;
        }
    }
    return {(int)room, smem};
}

template <typename IT, typename OT, bool kWide, int C>
cudaError_t launch_sized(const LogitArgs& a, size_t max_smem, cudaStream_t stream)
{
    auto kern = logits_kernel<IT, OT, kWide, C>;
    const Plan s = plan<kWide, C>(a, max_smem);
    static thread_local bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(max_smem - kStaticSmem));
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.M * C));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, a, s.room);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename IT, typename OT>
cudaError_t launch_typed(const LogitArgs& a, int num_sms, size_t max_smem, cudaStream_t stream)
{
    const bool wide = (a.history && a.history_count > 32767) || (a.bias_ids && a.bias_count > 65534);
    // Eight CTAs a row while they all find room at a time, and where four would be too large for two to an SM
    // (64 rows of 152064 with histories of 4096 and 300 biases: 36 us, with four 42; without biases 32 and 27).
    const bool eight = a.M * 8 <= (size_t)num_sms * 2 ||
                       (wide ? plan<true, 4>(a, max_smem) : plan<false, 4>(a, max_smem)).smem > 112 * 1024;
    if (wide)
        return eight ? launch_sized<IT, OT, true, 8>(a, max_smem, stream) : launch_sized<IT, OT, true, 4>(a, max_smem, stream);
    return eight ? launch_sized<IT, OT, false, 8>(a, max_smem, stream) : launch_sized<IT, OT, false, 4>(a, max_smem, stream);
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
