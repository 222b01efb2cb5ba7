// The operators of fl_ops.cu as the models' own paths call them (arguments as the C ABI checks them there).
#pragma once
#include "../../include/fastllm_b200.h"
#include "runtime.cuh"

namespace fl {

// 8-bit rows start on 16-byte borders
inline int64_t padded8(int64_t k) { return (k + 15) / 16 * 16; }
size_t linear8_workspace(int64_t rows, int64_t k);              // bytes (0: none is needed), no less than of fewer rows; the workspace starts on a 256-byte border
void op_quantize_rows(LaunchCtx& lc, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale);
// y = f32 [rows, n], x = f32 [rows, k], w = 8-bit [n, padded8(k)]; *failed is set when a wait in the kernel ran out (page-locked memory, see step_check)
void op_linear8(LaunchCtx& lc, const float* x, const int8_t* w, const float* w_scale, int64_t rows, int64_t n, int64_t k, float* y, void* workspace, size_t workspace_bytes, int* failed);
// logits f32 [rows, vocab], tokens [rows, given]; all pointers device memory
void op_logprobs(LaunchCtx& lc, const float* logits, int64_t rows, int64_t vocab, const int32_t* tokens, int64_t given, double temperature, int top, float* logprob,
                 float* logsumexp, float* entropy, int32_t* top_ids, float* top_logprobs);

}  // namespace fl
