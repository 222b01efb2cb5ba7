// Operators on device memory: argument checks and launches behind the C ABI (include/fastllm_b200.h, "operators on device memory").
#include <cmath>

#include "../../include/fastllm_b200.h"
#include "linear8.cuh"
#include "logprobs.cuh"
#include "runtime.cuh"

namespace fl {

// The bound device for the length of a call; the caller's own is put back.
struct DeviceScope {
    int before = -1, now;
    DeviceScope() : now(bound_device()) {
        FL_CUDA(cudaGetDevice(&before));
        if (before != now) FL_CUDA(cudaSetDevice(now));
    }
    ~DeviceScope() { if (before >= 0 && before != now) cudaSetDevice(before); }
};

static LaunchCtx op_ctx(void* stream) {
    LaunchCtx lc;
    lc.stream = static_cast<cudaStream_t>(stream);
    lc.pdl = false;
    if (g_prof.on) {                        // (no events inside a caller's capture)
        cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
        FL_CUDA(cudaStreamIsCapturing(lc.stream, &st));
        lc.capturing = st != cudaStreamCaptureStatusNone;
    }
    return lc;
}
static size_t dtype_size(int dtype) { return dtype == FL_DTYPE_F32 ? 4 : dtype == FL_DTYPE_I8 ? 1 : 2; }
static bool is_float(int dtype) { return dtype == FL_DTYPE_F32 || dtype == FL_DTYPE_BF16 || dtype == FL_DTYPE_F16; }
static bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxRows = (int64_t)1 << 30;
constexpr int64_t kLinear8MaxK = 131071;        // 128 * 128 * k stays below 2^31

static int64_t padded_k(int64_t k) { return (k + 15) / 16 * 16; }
static size_t quantized_bytes(int64_t rows, int64_t k) { return ((size_t)rows * padded_k(k) + 255) / 256 * 256; }

static void quantize_rows(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, int64_t cols_q, float* scale) {
    auto go = [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        launch(lc, "quantize_rows", rows * cols * (sizeof(T) + 1), quantize_rows_kernel<T>, dim3((unsigned)rows), dim3(256), 0, static_cast<const T*>(x), (long long)ldx,
               (int)cols, q, (long long)ldq, (int)cols_q, scale);
    };
    if (dtype == FL_DTYPE_F32) go((float*)nullptr);
    else if (dtype == FL_DTYPE_BF16) go((__nv_bfloat16*)nullptr);
    else go((__half*)nullptr);
}

}  // namespace fl

using namespace fl;

extern "C" {

FL_EXPORT int fl_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "quantize_rows: rows of f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kLinear8MaxK, FL_ERR_INVALID, "quantize_rows: rows from 0 to 2^30, columns from 1 to 131071");
    FL_CHECK(rows <= 1 || (ldx >= cols && ldq >= cols), FL_ERR_INVALID, "quantize_rows: a row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && q && scale, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(x, dtype_size(dtype)) && aligned(scale, 4), FL_ERR_INVALID, "quantize_rows: a pointer is not aligned to its type");
    DeviceScope dev;
    LaunchCtx lc = op_ctx(stream);
    quantize_rows(lc, x, dtype, rows, cols, ldx, q, ldq, cols, scale);
    FL_API_END
}

FL_EXPORT int fl_linear8_workspace(int64_t rows, int64_t k, int x_dtype, size_t* bytes) {
    FL_API_BEGIN
    FL_CHECK(bytes, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(is_float(x_dtype) || x_dtype == FL_DTYPE_I8, FL_ERR_INVALID, "linear8: activations are f32, bf16, f16 or i8");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && k >= 1 && k <= kLinear8MaxK, FL_ERR_INVALID, "linear8: rows from 0 to 2^30, k from 1 to 131071");
    *bytes = x_dtype == FL_DTYPE_I8 ? 0 : quantized_bytes(rows, k) + (size_t)rows * 4;
    FL_API_END
}

FL_EXPORT int fl_linear8(const void* x, int x_dtype, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias,
                         int64_t rows, int64_t n, int64_t k, void* y, int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    FL_API_BEGIN
    const bool given = x_dtype == FL_DTYPE_I8;
    FL_CHECK(is_float(x_dtype) || given, FL_ERR_INVALID, "linear8: activations are f32, bf16, f16 or i8");
    FL_CHECK(is_float(y_dtype), FL_ERR_INVALID, "linear8: results are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && n >= 1 && n <= kMaxRows && k >= 1 && k <= kLinear8MaxK, FL_ERR_INVALID,
             "linear8: rows from 0 to 2^30, n from 1 to 2^30, k from 1 to 131071");
    FL_CHECK((rows <= 1 || (ldx >= k && ldy >= n)) && (n == 1 || ldw >= k), FL_ERR_INVALID, "linear8: a row stride is smaller than the row");
    if (rows == 0) return FL_OK;
    FL_CHECK(x && w && w_scale && y, FL_ERR_INVALID, "NULL argument");
    FL_CHECK(given == (x_scale != nullptr), FL_ERR_INVALID, "linear8: x_scale comes with activations of 8 bits, and only with them");
    FL_CHECK(aligned(w, 16) && (n == 1 || ldw % 16 == 0), FL_ERR_INVALID, "linear8: the weight's rows start on 16-byte borders (pointer and row stride)");
    FL_CHECK(!given || (aligned(x, 16) && (rows == 1 || ldx % 16 == 0)), FL_ERR_INVALID, "linear8: 8-bit activation rows start on 16-byte borders (pointer and row stride)");
    FL_CHECK(aligned(x, dtype_size(x_dtype)) && aligned(y, dtype_size(y_dtype)) && aligned(w_scale, 4) && aligned(x_scale, 4) && aligned(bias, 4), FL_ERR_INVALID,
             "linear8: a pointer is not aligned to its type");
    const size_t need = given ? 0 : quantized_bytes(rows, k) + (size_t)rows * 4;
    FL_CHECK(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), FL_ERR_INVALID,
             "linear8: the workspace is smaller than fl_linear8_workspace asks for, or not on a 256-byte border");
    DeviceScope dev;
    LaunchCtx lc = op_ctx(stream);
    Linear8Args g{};
    if (given) {
        g.xq = static_cast<const int8_t*>(x); g.ldq = ldx; g.xs = x_scale;
    } else {
        int8_t* q = static_cast<int8_t*>(workspace);
        float* s = reinterpret_cast<float*>(q + quantized_bytes(rows, k));
        quantize_rows(lc, x, x_dtype, rows, k, ldx, q, padded_k(k), padded_k(k), s);
        g.xq = q; g.ldq = padded_k(k); g.xs = s;
    }
    g.w = w; g.ldw = ldw; g.ws = w_scale; g.bias = bias; g.y = y; g.ldy = ldy;
    g.rows = (int)rows; g.n = (int)n; g.k = (int)k;
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((rows + 63) / 64));
    FL_CHECK(grid.y <= 65535, FL_ERR_INVALID, "linear8: too many rows");
    const uint64_t bytes = (uint64_t)n * k + (uint64_t)rows * (k + n * dtype_size(y_dtype));
    if (y_dtype == FL_DTYPE_F32) launch(lc, "linear8", bytes, linear8_kernel<float>, grid, dim3(256), 0, g);
    else if (y_dtype == FL_DTYPE_BF16) launch(lc, "linear8", bytes, linear8_kernel<__nv_bfloat16>, grid, dim3(256), 0, g);
    else launch(lc, "linear8", bytes, linear8_kernel<__half>, grid, dim3(256), 0, g);
    FL_API_END
}

FL_EXPORT int fl_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* tokens, int token_bytes, int64_t given,
                          double temperature, int top, float* logprob, float* logsumexp, float* entropy, int32_t* top_ids, float* top_logprobs, void* stream) {
    FL_API_BEGIN
    FL_CHECK(is_float(dtype), FL_ERR_INVALID, "logprobs: logits are f32, bf16 or f16");
    FL_CHECK(rows >= 0 && rows <= kMaxRows && vocab >= 1 && vocab <= kLpMaxVocab, FL_ERR_INVALID, "logprobs: rows from 0 to 2^30, a vocabulary from 1 to 2^20");
    FL_CHECK(rows <= 1 || ld >= vocab, FL_ERR_INVALID, "logprobs: the row stride is smaller than the vocabulary");
    FL_CHECK(given >= 0 && given <= kLpMaxVocab && (given == 0 || token_bytes == 4 || token_bytes == 8), FL_ERR_INVALID, "logprobs: given tokens are 32- or 64-bit integers");
    FL_CHECK(top >= 0 && top <= kLpMaxTop && top <= vocab, FL_ERR_INVALID, "logprobs: from 0 to 32 alternatives, and no more than the vocabulary has");
    const float inv_t = (float)(1.0 / temperature);
    FL_CHECK(temperature > 0 && std::isfinite(temperature) && std::isfinite(inv_t) && inv_t > 0, FL_ERR_INVALID, "logprobs: the temperature is a positive number");
    if (rows == 0) return FL_OK;
    FL_CHECK(logits && (given == 0 || (tokens && logprob)) && (top == 0 || (top_ids && top_logprobs)), FL_ERR_INVALID, "NULL argument");
    FL_CHECK(aligned(logits, dtype_size(dtype)) && (given == 0 || aligned(tokens, token_bytes)) && aligned(logprob, 4) && aligned(logsumexp, 4) && aligned(entropy, 4) &&
                 aligned(top_ids, 4) && aligned(top_logprobs, 4), FL_ERR_INVALID, "logprobs: a pointer is not aligned to its type");
    DeviceScope dev;
    LaunchCtx lc = op_ctx(stream);
    const LogprobArgs a{logits, ld, (int)rows, (int)vocab, inv_t, tokens, (int)given, token_bytes == 8, top, given ? logprob : nullptr, logsumexp, entropy, top_ids, top_logprobs};
    const uint64_t bytes = (uint64_t)rows * vocab * dtype_size(dtype);
    const dim3 grid((unsigned)rows);
    if (dtype == FL_DTYPE_F32) launch(lc, "logprobs", bytes, logprobs_kernel<float>, grid, dim3(256), 0, a);
    else if (dtype == FL_DTYPE_BF16) launch(lc, "logprobs", bytes, logprobs_kernel<__nv_bfloat16>, grid, dim3(256), 0, a);
    else launch(lc, "logprobs", bytes, logprobs_kernel<__half>, grid, dim3(256), 0, a);
    FL_API_END
}

}  // extern "C"
