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
// A cluster of CTAs serves one row: each CTA owns a slice of the vocabulary, counts the history's
// tokens of its slice in shared memory (integer atomics, so the order does not matter), then passes
// over its logits once.  The CTAs' best tokens meet in the first CTA's shared memory.  No workspace.
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

constexpr int kLogitThreads = 512;
constexpr int kLogitCluster = 8;
constexpr uint32_t kInPrompt = 0x80000000u;  // the token is in the prompt; the other bits count the output

// Unsigned key of a float that is no NaN: larger value, larger key; -0 and +0 alike.
__device__ __forceinline__ uint32_t order_key(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A thread's view of the greedy choice: `best` = (key of the value, complement of the token), so the
// first of equal values wins; `first` = the first candidate * 2 + (it is NaN).  NaN candidates lose
// to any number; the first candidate wins if it is NaN (std::max_element's order).
struct Best {
    unsigned long long best = 0, first = ~0ull;
    __device__ __forceinline__ void take(float v, uint32_t i)
    {
        const bool nan = v != v;
        const unsigned long long f = ((unsigned long long)i << 1) | (nan ? 1u : 0u);
        first = f < first ? f : first;
        const unsigned long long k = nan ? 0ull : ((unsigned long long)order_key(v) << 32) | (uint32_t)~i;
        best = k > best ? k : best;
    }
    __device__ __forceinline__ void merge(unsigned long long b, unsigned long long f)
    {
        best = b > best ? b : best;
        first = f < first ? f : first;
    }
    __device__ __forceinline__ int token() const
    {
        if (first == ~0ull) return -1;
        return (first & 1) ? (int)(first >> 1) : (int)~(uint32_t)best;
    }
};

template <typename IT, typename OT>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitArgs a, int slice)
{
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long m = blockIdx.x / C;
    const int tid = threadIdx.x;
    extern __shared__ uint32_t smem[];
    __shared__ unsigned long long red[2][kLogitThreads / 32], joined[2][16];

    const int V = (int)a.V;
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
    const IT* in = static_cast<const IT*>(a.logits) + m * (long long)a.in_stride;
    OT* out = a.out ? static_cast<OT*>(a.out) + m * (long long)a.out_stride : nullptr;
    uint32_t* count = smem;
    int* entry = reinterpret_cast<int*>(smem + (a.history ? slice : 0));  // 1 + a token's last bias entry, or 0

    Best b;
    for (long long base = (long long)rank * slice; base < V; base += (long long)C * slice) {
        const int n = (int)min((long long)slice, V - base);
        for (int i = tid; i < n; i += kLogitThreads) {
            if (hlen) count[i] = 0;
            if (blen) entry[i] = 0;
        }
        __syncthreads();
        for (int j = tid; j < hlen; j += kLogitThreads) {
            const long long u = (long long)hist[j] - base;
            if (u >= 0 && u < n) {
                if (j < plen)
                    atomicOr(count + u, kInPrompt);
                else
                    atomicAdd(count + u, 1u);
            }
        }
        for (int j = tid; j < blen; j += kLogitThreads) {
            const long long u = (long long)bids[j] - base;
            if (u >= 0 && u < n) atomicMax(entry + u, j + 1);
        }
        __syncthreads();
        for (int i = tid; i < n; i += kLogitThreads) {
            const int tok = (int)base + i;
            float v = load_as_f32<IT>(in + tok);
            const uint32_t c = hlen ? count[i] : 0u;
            if (c) {
                v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                const uint32_t made = c & ~kInPrompt;
                if (made) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)made)), pres);
            }
            const int e = blen ? entry[i] : 0;
            if (e) v = __fadd_rn(v, bval[e - 1]);
            const bool ok = !mask || ((mask[tok >> 5] >> (tok & 31)) & 1u);
            if (!ok) v = -INFINITY;
            OT o;
            store_from_f32<OT>(&o, v);
            if (out) out[tok] = o;
            if (ok) b.take(load_as_f32<OT>(&o), (uint32_t)tok);
        }
        __syncthreads();  // the counts are read; the next slice may clear them
    }
    if (!a.argmax) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        b.merge(__shfl_xor_sync(0xffffffffu, b.best, o), __shfl_xor_sync(0xffffffffu, b.first, o));
    if ((tid & 31) == 0) {
        red[0][tid >> 5] = b.best;
        red[1][tid >> 5] = b.first;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kLogitThreads / 32; w++) b.merge(red[0][w], red[1][w]);
        unsigned long long* to = cluster.map_shared_rank(&joined[0][0], 0);
        to[rank] = b.best;
        to[16 + rank] = b.first;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        Best all;
        for (int r = 0; r < C; r++) all.merge(joined[0][r], joined[1][r]);
        a.argmax[m] = all.token();
    }
}

template <typename IT, typename OT>
cudaError_t launch_typed(const LogitArgs& a, size_t max_smem, cudaStream_t stream)
{
    auto kern = logits_kernel<IT, OT>;
    const size_t words = (a.history ? 1 : 0) + (a.bias_ids ? 1 : 0);
    // A slice is whole mask words; what a CTA's counters may take is what is left beside the static part.
    long long slice = ((long long)a.V + kLogitCluster - 1) / kLogitCluster;
    slice = (slice + 31) / 32 * 32;
    if (words) slice = std::min<long long>(slice, (long long)((max_smem - 2048) / (4 * words)) / 32 * 32);
    const size_t smem = words * 4 * (size_t)slice;
    static thread_local bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(max_smem - 2048));
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.M * kLogitCluster));
    cfg.blockDim = dim3(kLogitThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kLogitCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, a, (int)slice);
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace

cudaError_t launch_logits(const LogitArgs& a, size_t max_smem, cudaStream_t stream)
{
    if (a.in_dtype == kF16)
        return a.out_dtype == kF16 ? launch_typed<__half, __half>(a, max_smem, stream)
                                   : launch_typed<__half, float>(a, max_smem, stream);
    return a.out_dtype == kF16 ? launch_typed<float, __half>(a, max_smem, stream)
                               : launch_typed<float, float>(a, max_smem, stream);
}

}  // namespace b200q8
