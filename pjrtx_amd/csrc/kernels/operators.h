// Launchers of the operator kernels (kernels/paged.hip, kernels/norm.hip,
// kernels/logprobs.hip): the custom calls of a decoder's serving and training
// step. Tensors are dense and row-major; no pointer needs more than its
// element's alignment.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.h"

namespace pjrtx {

// --------------------------------------------------------- paged attention

// out[b, h] = softmax_j(scale * q[b, h] . k_j) . v_j over the keys j of
// sequence b that are attended: lengths[b] - window <= j < lengths[b] (no
// lower bound when window is 0) and page_table[b, j / S] in [0, P). Key j's
// rows are k_pages / v_pages[page, h / (Hq / Hkv), j % S]. A sequence with no
// attended key answers zeros. lengths are read as at most M * S.
struct PagedParams {
  int64_t B = 0;
  int Hq = 0, Hkv = 0, D = 0;
  int64_t P = 0, S = 0, M = 0;
  int64_t window = 0;
  float scale = 1.f;
};
// Device scratch of the split lengths' partial results.
size_t paged_attention_scratch_bytes(const PagedParams& p, DType t);
void launch_paged_attention(hipStream_t s, const PagedParams& p, DType t, const void* q, const void* k_pages,
                            const void* v_pages, const int32_t* page_table, const int32_t* lengths, void* out,
                            void* scratch);

// k_pages / v_pages[slot / S, :, slot % S] = k_new / v_new[n] for slot =
// slots[n]; slots outside [0, P * S) are skipped, and of rows that name one
// slot the last stays.
struct AppendParams {
  int64_t N = 0, Hkv = 0, D = 0, P = 0, S = 0;
  int slot_bytes = 4;
};
void launch_paged_append(hipStream_t s, const AppendParams& p, int elem_bytes, void* k_pages, void* v_pages,
                         const void* k_new, const void* v_new, const void* slots);

// ------------------------------------------------------------ residual norm

// t = x + residual (x alone when residual is null); y = t * gain /
// sqrt(mean(t^2) + eps). `sum` (when set) receives t. Either y in the type t,
// or y8 = y / scale rounded to the nearest even with scales[row] =
// max|y| / 127.
struct NormParams {
  int64_t rows = 0, D = 0;
  float eps = 0.f;
};
void launch_add_rms_norm(hipStream_t s, const NormParams& p, DType t, const void* x, const void* residual,
                         const void* gain, void* y, int8_t* y8, float* scales, void* sum);

// dx = dsum + r (dn - n mean(dn n)), dgain = sum over the rows of dy n, with
// r = 1 / sqrt(mean(t^2) + eps), n = t r, dn = dy gain; dsum may be null.
size_t add_rms_norm_grad_scratch_bytes(const NormParams& p, DType t);
void launch_add_rms_norm_grad(hipStream_t s, const NormParams& p, DType t, const void* dy, const void* dsum,
                              const void* sum, const void* gain, void* dx, void* dgain, void* scratch);

// -------------------------------------------------- token log probabilities

// lse = log sum_j exp(x_j); logprob = x_token - lse (0 where the token is
// outside [0, V)); entropy = lse - sum_j p_j x_j; the top_k largest x_j - lse
// with their indices, in the order of top_k (ties to the lowest index).
struct LogprobsParams {
  int64_t rows = 0, V = 0;
  int top_k = 0;
  int token_bytes = 4;
};
constexpr int kLogprobsMaxTopK = 128;
size_t token_logprobs_scratch_bytes(const LogprobsParams& p, DType t);
void launch_token_logprobs(hipStream_t s, const LogprobsParams& p, DType t, const void* logits, const void* tokens,
                           float* logprobs, float* entropy, float* lse, float* top_logprobs, int32_t* top_tokens,
                           void* scratch);

// d_logits_j = d_logprob (1[j == token] - p_j) - d_entropy p_j (log p_j +
// entropy), p_j = exp(x_j - lse); d_logprob counts as 0 where the token is
// outside [0, V).
void launch_token_logprobs_grad(hipStream_t s, const LogprobsParams& p, DType t, const void* logits,
                                const void* tokens, const float* lse, const float* entropy, const float* d_logprobs,
                                const float* d_entropy, void* d_logits);

}  // namespace pjrtx
