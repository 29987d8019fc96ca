// q4_api.cu -- the extern "C" boundary of the 4-bit weights and of the logits step (include/b200q8.h).
#include <cuda_runtime.h>

#include <cstdint>

#include "b200q8.h"
#include "kernels.h"

namespace b200q8 {
namespace {

bool known_dtype(int d) { return d == B200Q8_F32 || d == B200Q8_F16; }
size_t elem_bytes(int d) { return d == B200Q8_F16 ? 2 : 4; }

bool overlap(const void* a, size_t na, const void* b, size_t nb)
{
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    return a0 < b0 + nb && b0 < a0 + na;
}

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Sizes of a 4-bit matrix; fails on a group or size it cannot have.
struct Q4Shape {
    size_t code_bytes = 0, scale_bytes = 0;
};
int q4_shape(const char* what, size_t N, size_t K, int group, Q4Shape* s)
{
    if (group != 32 && group != 64 && group != 128)
        return fail(B200Q8_ERR_INVALID, "%s: group must be 32, 64 or 128, got %d", what, group);
    if (K == 0) return fail(B200Q8_ERR_INVALID, "%s: K == 0", what);
    if (N > (size_t)INT32_MAX || K > (size_t)INT32_MAX)
        return fail(B200Q8_ERR_INVALID, "%s: sizes overflow (N=%zu K=%zu)", what, N, K);
    s->code_bytes = N * ((K + 1) / 2);
    s->scale_bytes = N * ((K + group - 1) / group) * 2;
    return B200Q8_OK;
}

int quantize_q4(const char* what, const void* w, int w_bf16, size_t N, size_t K, int group, uint8_t* q4,
                uint16_t* scales, cudaStream_t stream)
{
    Q4Shape s;
    int st = q4_shape(what, N, K, group, &s);
    if (st) return st;
    if (N == 0) return B200Q8_OK;
    if (!w || !q4 || !scales) return fail(B200Q8_ERR_INVALID, "%s: null pointer", what);
    const size_t wb = N * K * (w_bf16 ? 2 : 4);
    if (!aligned(w, w_bf16 ? 2 : 4) || !aligned(scales, 2))
        return fail(B200Q8_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    if (overlap(w, wb, q4, s.code_bytes) || overlap(w, wb, scales, s.scale_bytes) ||
        overlap(q4, s.code_bytes, scales, s.scale_bytes))
        return fail(B200Q8_ERR_INVALID, "%s: w, q4 and scales overlap", what);
    int sms = 0;
    size_t smem = 0;
    if ((st = current_device(&sms, &smem))) return st;
    cudaError_t e = launch_q4_quantize(w, w_bf16, N, K, group, q4, scales, sms, stream);
    return e == cudaSuccess ? B200Q8_OK : cuda_fail(e, "q4_quantize launch");
}

int linear_q4(const char* what, void* out, int out_dtype, const void* inp, int in_dtype, const uint8_t* q4,
              const uint16_t* scales, int group, const float* bias, const void* residual, size_t M, size_t N, size_t K,
              cudaStream_t stream)
{
    if (!known_dtype(out_dtype) || !known_dtype(in_dtype))
        return fail(B200Q8_ERR_INVALID, "%s: dtype must be B200Q8_F32 or B200Q8_F16", what);
    Q4Shape s;
    int st = q4_shape(what, N, K, group, &s);
    if (st) return st;
    if (M > (size_t)INT32_MAX) return fail(B200Q8_ERR_INVALID, "%s: sizes overflow (M=%zu)", what, M);
    if (M == 0 || N == 0) return B200Q8_OK;
    if (!out || !inp || !q4 || !scales) return fail(B200Q8_ERR_INVALID, "%s: null out/inp/q4/scales", what);
    const size_t ob = elem_bytes(out_dtype), ib = elem_bytes(in_dtype);
    if (!aligned(out, ob) || !aligned(inp, ib) || !aligned(scales, 2) || !aligned(bias, 4) || !aligned(residual, ob))
        return fail(B200Q8_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const size_t on = M * N * ob;
    if (overlap(out, on, inp, M * K * ib)) return fail(B200Q8_ERR_INVALID, "%s: inp overlaps out", what);
    if (overlap(out, on, q4, s.code_bytes) || overlap(out, on, scales, s.scale_bytes))
        return fail(B200Q8_ERR_INVALID, "%s: the weights overlap out", what);
    if (bias && overlap(out, on, bias, N * 4)) return fail(B200Q8_ERR_INVALID, "%s: bias overlaps out", what);
    if (residual && residual != out && overlap(out, on, residual, on))
        return fail(B200Q8_ERR_INVALID, "%s: residual partially overlaps out", what);
    int sms = 0;
    size_t smem = 0;
    if ((st = current_device(&sms, &smem))) return st;
    Q4Args a;
    a.x = inp;
    a.q4 = q4;
    a.scales = scales;
    a.bias = bias;
    a.res = residual;
    a.out = out;
    a.M = M;
    a.N = N;
    a.K = K;
    a.group = group;
    a.in_dtype = in_dtype;
    a.out_dtype = out_dtype;
    // The streaming kernel goes over the weights once for every 16 fp16 tokens (8 in fp32), in passes that run side by
    // side; the GEMM (fp16 tokens) once, bound by its dequantization at 64 tokens and with a start of its own.
    // Measured on B200, streaming vs GEMM: 37888 x 3584 at 16 tokens 24 vs 38 us, at 17 39 vs 38; 3584 x 3584 at 64 16
    // vs 21, at 128 25 vs 24; 896 x 4864 at 64 12 vs 26, at 256 26 vs 25; 4864 x 896 at 32 9 vs 10, at 64 11 vs 10.
    // With K of a few hundred the rule takes the GEMM too early: 37888 x 256 at 32 9 vs 13, x 512 11 vs 14; 9600 x 256 at
    // 300 16 vs 23, x 128 18 vs 22.
    // Up to 16 tokens only those that need clusters of eight are slower: 3584 x 18944 at 9 24 vs 28, at 16 38 vs 28;
    // 8192 x 28672 at 8 38 vs 64, at 9 72 vs 64.
    const size_t work = M * N * K;
    bool gemm = M > 16 ? work > (K < 2048 ? (size_t)1 << 28 : (size_t)1 << 30) : M > 8 && M * K > 200 * 1024 && work > ((size_t)1 << 29);
    // fp32 outputs take the GEMM only with short sums: the tensor core's accumulator drops what falls below its 24
    // bits instead of rounding it, 1.8e-8 of the sum per 16 products (512 tokens, K = 18944: 2.2e-5 off, where
    // fp32 sums in another order are 2e-6 off and the streaming kernel's 3e-7); half an fp16 step is 2^-12.
    gemm = gemm && (out_dtype == B200Q8_F16 || K <= 512);
    // Rows that the fast kernels do not take are copied into ones that they do, but for the small: then the generic
    // kernel is as quick as the copies' launches (1 x 896 x 255 4.7 us, copied 5.8; 4 x 896 x 255 6.9, 6.0; 100 x 300 x 77
    // 6.2, 13; 1 x 896 x 895 9.8, 6.4; 512 x 3584 x 3583 4611, 43).
    const bool small = (K < 192 || K * (M < 8 ? M : 8) < 768) && work < ((size_t)1 << 23);
    const size_t pad = small ? 0 : q4_pad_bytes(a);
    Q4Args fast = a;  // as it will be after the copying
    if (pad) fast.q4 = nullptr, fast.x = nullptr, fast.K = (K + 31) / 32 * 32;
    const bool use_gemm = gemm && q4_gemm_tc_supports(fast);
    ScratchHold hold;  // to the last launch below
    if (use_gemm || pad) {
        size_t ws = 0, counters = 0, act = 0;
        if (use_gemm) q4_gemm_tc_scratch_need(fast, sms, &ws, &counters, &act);
        act = (act + 255) / 256 * 256;
        TcScratch scratch;
        if ((st = stream_scratch(ws, counters, act + pad, sms, stream, &hold, &scratch))) return st;
        cudaError_t e = pad ? launch_q4_pad(&a, scratch.act + act, sms, stream) : cudaSuccess;
        if (e != cudaSuccess) return cuda_fail(e, "q4_pad launch");
        if (use_gemm) {
            e = launch_q4_gemm_tc(a, sms, scratch, stream);
            return e == cudaSuccess ? B200Q8_OK : cuda_fail(e, "q4_gemm launch");
        }
    }
    cudaError_t e = launch_q4_stream(a, sms, smem, stream);
    if (e == cudaErrorNotSupported) e = launch_q4_linear_generic(a, stream);
    return e == cudaSuccess ? B200Q8_OK : cuda_fail(e, "q4_linear launch");
}

}  // namespace
}  // namespace b200q8

using namespace b200q8;

extern "C" {

int b200q8_quantize_q4(const float* w, size_t N, size_t K, int group, uint8_t* q4, uint16_t* scales,
                       b200q8_stream_t stream)
{
    return quantize_q4("quantize_q4", w, 0, N, K, group, q4, scales, (cudaStream_t)stream);
}

int b200q8_quantize_q4_bf16(const uint16_t* w, size_t N, size_t K, int group, uint8_t* q4, uint16_t* scales,
                            b200q8_stream_t stream)
{
    return quantize_q4("quantize_q4_bf16", w, 1, N, K, group, q4, scales, (cudaStream_t)stream);
}

int b200q8_dequantize_q4(void* out, int out_dtype, const uint8_t* q4, const uint16_t* scales, int group,
                         const int32_t* rows, size_t R, size_t N, size_t K, b200q8_stream_t stream)
{
    const char* what = "dequantize_q4";
    if (!known_dtype(out_dtype)) return fail(B200Q8_ERR_INVALID, "%s: dtype must be B200Q8_F32 or B200Q8_F16", what);
    Q4Shape s;
    int st = q4_shape(what, N, K, group, &s);
    if (st) return st;
    if (!rows && R != N) return fail(B200Q8_ERR_INVALID, "%s: without rows, R must be N (R=%zu N=%zu)", what, R, N);
    if (R > (size_t)INT32_MAX) return fail(B200Q8_ERR_INVALID, "%s: sizes overflow (R=%zu)", what, R);
    if (R == 0) return B200Q8_OK;
    if (!out || (N && (!q4 || !scales))) return fail(B200Q8_ERR_INVALID, "%s: null pointer", what);
    const size_t ob = elem_bytes(out_dtype), on = R * K * ob;
    if (!aligned(out, ob) || !aligned(scales, 2) || !aligned(rows, 4))
        return fail(B200Q8_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    if (overlap(out, on, q4, s.code_bytes) || overlap(out, on, scales, s.scale_bytes) ||
        (rows && overlap(out, on, rows, R * 4)))
        return fail(B200Q8_ERR_INVALID, "%s: out overlaps an input", what);
    int sms = 0;
    size_t smem = 0;
    if ((st = current_device(&sms, &smem))) return st;
    cudaError_t e = launch_q4_dequantize(out, out_dtype, q4, scales, group, rows, R, N, K, sms, (cudaStream_t)stream);
    return e == cudaSuccess ? B200Q8_OK : cuda_fail(e, "q4_dequantize launch");
}

int b200q8_linear_q4(void* out, int out_dtype, const void* inp, int in_dtype, const uint8_t* q4, const uint16_t* scales,
                     int group, const float* bias, size_t M, size_t N, size_t K, b200q8_stream_t stream)
{
    return linear_q4("linear_q4", out, out_dtype, inp, in_dtype, q4, scales, group, bias, nullptr, M, N, K,
                     (cudaStream_t)stream);
}

int b200q8_linear_q4_add(void* out, int out_dtype, const void* inp, int in_dtype, const uint8_t* q4,
                         const uint16_t* scales, int group, const float* bias, const void* residual, size_t M, size_t N,
                         size_t K, b200q8_stream_t stream)
{
    return linear_q4("linear_q4_add", out, out_dtype, inp, in_dtype, q4, scales, group, bias, residual, M, N, K,
                     (cudaStream_t)stream);
}

int b200q8_process_logits(void* out, int out_dtype, size_t out_stride, const void* logits, int in_dtype,
                          size_t in_stride, size_t M, size_t V, const b200q8_logit_rules* rules, int32_t* argmax,
                          b200q8_stream_t stream)
{
    const char* what = "process_logits";
    if (!known_dtype(out_dtype) || !known_dtype(in_dtype))
        return fail(B200Q8_ERR_INVALID, "%s: dtype must be B200Q8_F32 or B200Q8_F16", what);
    const b200q8_logit_rules none = {};
    const b200q8_logit_rules& r = rules ? *rules : none;
    constexpr size_t kMax = (size_t)INT32_MAX;
    if (M > kMax / 16 || V > kMax - 65536 || r.history_count > kMax || r.bias_count > kMax - 1)
        return fail(B200Q8_ERR_INVALID, "%s: sizes overflow (M=%zu V=%zu)", what, M, V);
    if (M == 0) return B200Q8_OK;
    if (V == 0) return fail(B200Q8_ERR_INVALID, "%s: V == 0", what);
    if (!logits || (!out && !argmax)) return fail(B200Q8_ERR_INVALID, "%s: null logits, or neither out nor argmax", what);
    constexpr size_t kMaxStride = (size_t)1 << 40;
    if (r.history_stride > kMaxStride || r.bias_stride > kMaxStride || r.allowed_stride > kMaxStride ||
        in_stride > kMaxStride || out_stride > kMaxStride)
        return fail(B200Q8_ERR_INVALID, "%s: a stride overflows", what);
    if (in_stride < V || (out && out_stride < V))
        return fail(B200Q8_ERR_INVALID, "%s: logits and out rows must not overlap (strides below V=%zu)", what, V);
    if (r.history && !r.history_len) return fail(B200Q8_ERR_INVALID, "%s: history needs history_len", what);
    if ((r.bias_ids == nullptr) != (r.bias_values == nullptr))
        return fail(B200Q8_ERR_INVALID, "%s: bias_ids and bias_values come together", what);
    const size_t words = (V + 31) / 32;
    if ((r.history && r.history_stride && r.history_stride < r.history_count) ||
        (r.bias_ids && r.bias_stride && r.bias_stride < r.bias_count) ||
        (r.allowed && r.allowed_stride && r.allowed_stride < words))
        return fail(B200Q8_ERR_INVALID, "%s: a row of history, biases or allowed is longer than its stride", what);
    const size_t ib = elem_bytes(in_dtype), ob = elem_bytes(out_dtype);
    const void* fours[] = {argmax, r.history, r.history_len, r.prompt_len, r.repetition, r.presence, r.frequency,
                           r.bias_ids, r.bias_values, r.bias_len, r.allowed};
    for (const void* p : fours)
        if (!aligned(p, 4)) return fail(B200Q8_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    if (!aligned(logits, ib) || !aligned(out, ob))
        return fail(B200Q8_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const size_t in_bytes = ((M - 1) * in_stride + V) * ib, out_bytes = out ? ((M - 1) * out_stride + V) * ob : 0;
    const bool in_place = out == logits && in_dtype == out_dtype && in_stride == out_stride;
    if (out && !in_place && overlap(out, out_bytes, logits, in_bytes))
        return fail(B200Q8_ERR_INVALID, "%s: out overlaps logits", what);
    if (argmax && (overlap(argmax, M * 4, logits, in_bytes) || (out && overlap(argmax, M * 4, out, out_bytes))))
        return fail(B200Q8_ERR_INVALID, "%s: argmax overlaps logits or out", what);
    // What a row of the rules reads must not be what the call writes.
    const struct {
        const void* p;
        size_t n;
    } reads[] = {{r.history, r.history ? ((M - 1) * r.history_stride + r.history_count) * 4 : 0},
                 {r.history_len, M * 4},
                 {r.prompt_len, M * 4},
                 {r.repetition, M * 4},
                 {r.presence, M * 4},
                 {r.frequency, M * 4},
                 {r.bias_ids, r.bias_ids ? ((M - 1) * r.bias_stride + r.bias_count) * 4 : 0},
                 {r.bias_values, r.bias_ids ? ((M - 1) * r.bias_stride + r.bias_count) * 4 : 0},
                 {r.bias_len, M * 4},
                 {r.allowed, r.allowed ? ((M - 1) * r.allowed_stride + words) * 4 : 0}};
    for (const auto& x : reads)
        if (x.p && ((out && overlap(x.p, x.n, out, out_bytes)) || (argmax && overlap(x.p, x.n, argmax, M * 4))))
            return fail(B200Q8_ERR_INVALID, "%s: out or argmax overlaps an input", what);
    int sms = 0;
    size_t smem = 0;
    int st = current_device(&sms, &smem);
    if (st) return st;
    LogitArgs a;
    a.out = out;
    a.logits = logits;
    a.argmax = argmax;
    a.M = M;
    a.V = V;
    a.in_stride = in_stride;
    a.out_stride = out_stride;
    a.in_dtype = in_dtype;
    a.out_dtype = out_dtype;
    a.history = r.history;
    a.history_len = r.history_len;
    a.prompt_len = r.prompt_len;
    a.history_stride = r.history_stride;
    a.history_count = r.history_count;
    a.repetition = r.repetition;
    a.presence = r.presence;
    a.frequency = r.frequency;
    a.bias_ids = r.bias_ids;
    a.bias_values = r.bias_values;
    a.bias_len = r.bias_len;
    a.bias_stride = r.bias_stride;
    a.bias_count = r.bias_count;
    a.allowed = r.allowed;
    a.allowed_stride = r.allowed_stride;
    cudaError_t e = launch_logits(a, sms, smem, (cudaStream_t)stream);
    return e == cudaSuccess ? B200Q8_OK : cuda_fail(e, "process_logits launch");
}

}  // extern "C"
