// training.h -- table lookup, token log-probabilities, preference and policy
// losses, each with its gradient (host launchers).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sinkslot {

// Element types of tables, logits and their gradients.
enum DType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

inline int dtype_bytes(int dt) { return dt == kF32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }

// ---- lookup.cu -------------------------------------------------------------
int lookup(const void* table, int dtype, int64_t stride, int64_t rows, int64_t dim,
           const void* index, int index_bytes, int64_t count, double scale, void* out,
           cudaStream_t st);
size_t lookup_grad_workspace_bytes(int64_t count, int64_t rows, int64_t dim);
int lookup_grad(const void* grad_out, int dtype, int64_t stride, const void* index,
                int index_bytes, int64_t count, int64_t rows, int64_t dim, double scale,
                int64_t padding, void* grad_table, void* ws, size_t ws_bytes, cudaStream_t st);

// ---- logprobs.cu -----------------------------------------------------------
// log2(e) / T and 1 / T, each as the sum of two floats; the difference of two logits
// from which on the exponential is 0.
struct Scale2 {
  float hi = 0.0f, lo = 0.0f, inv = 0.0f, inv_lo = 0.0f, low = 0.0f;
};
// Rows of logits and the token chosen in each.
struct LogitRows {
  const void* z = nullptr;
  int dtype = 0;
  int64_t stride = 0;  // elements from one row to the next
  int64_t rows = 0, vocab = 0;
  const void* tokens = nullptr;
  int token_bytes = 8;
  int64_t ignore = 0;        // token value of a row that is left out
  const uint8_t* mask = nullptr;  // nullable: 0 leaves a row out as well
  double inv_temp = 1.0;
  Scale2 scale;  // set by token_logprobs
};
int check_rows(const LogitRows& r);
int token_logprobs(const LogitRows& r, float* logp, float* entropy, float2* stats,
                   cudaStream_t st);
// g, g_entropy: outer gradients (nullable), their strides in elements (0: one
// value for all); scale_dev, scale: factors of both.
struct LogitGrad {
  const float* g = nullptr;
  int64_t g_stride = 0;
  const float* g_entropy = nullptr;
  int64_t g_entropy_stride = 0;
  const float* scale_dev = nullptr;
  float scale = 1.0f;
  const float* entropy = nullptr;
  const float2* stats = nullptr;
  void* dz = nullptr;
  int64_t dz_stride = 0;
};
int token_logprobs_grad(const LogitRows& r, const LogitGrad& g, cudaStream_t st);

// ---- losses.cu -------------------------------------------------------------
// Packed sequences of tokens: sequence i holds [offsets[i], offsets[i + 1]).
struct Packed {
  int64_t tokens = 0;
  const void* offsets = nullptr;  // count + 1 values; null: one sequence of all tokens
  int offset_bytes = 8;
  int64_t count = 1;
  const uint8_t* mask = nullptr;  // nullable: 0 leaves a token out
};
struct PolicyTerms {
  const float* logp = nullptr;
  const float* old_logp = nullptr;
  const float* ref_logp = nullptr;  // nullable: no KL term
  const float* adv = nullptr;
  int adv_per_token = 0;
  double clip_low = 0, clip_high = 0, kl_coef = 0;
  int kl_kind = 3;           // 1, 2, 3
  int sequence_average = 0;  // 0: mean over tokens, 1: mean of the sequences' means
};
// What a row's gradient needs of the whole batch: the sequence of each token (-1:
// none), the sequences' counted tokens, and one over what the loss is averaged by.
struct PolicyRows {
  const int* owner = nullptr;
  const int64_t* counts = nullptr;
  const float* norm = nullptr;
};
// ---- policy_rows.cu: all rows' log-probabilities and gradient in one pass.
bool policy_rows_fit(const LogitRows& r, const void* dz, int64_t dz_stride);
int policy_rows(const LogitRows& r, const PolicyTerms& t, const PolicyRows& w, float grad_scale,
                float* logp, void* dz, int64_t dz_stride, cudaStream_t st);
struct PreferenceTerms {
  const float* logp = nullptr;
  const float* ref_logp = nullptr;  // nullable
  double beta = 0, smoothing = 0;
  int kind = 0;  // 0 sigmoid, 1 hinge, 2 squared
  int normalize = 0;
};
size_t loss_workspace_bytes(int64_t count);
// values[0..3] = loss, kl, clipped share, norm: the gradient of token t is
// coef[t] * norm.  coef nullable.
int policy_loss(const Packed& p, const PolicyTerms& t, float* values, float* coef, void* ws,
                size_t ws_bytes, cudaStream_t st);
// rewards[0..count): chosen, then rejected; slope[i]: gradient of every counted
// token of sequence i.
int preference_loss(const Packed& p, const PreferenceTerms& t, float* loss, float* rewards,
                    float* slope, void* ws, size_t ws_bytes, cudaStream_t st);
int preference_grad(const Packed& p, const float* slope, const float* g, float* out,
                    cudaStream_t st);
int scale_tokens(const float* coef, int64_t tokens, const float* norm, const float* g, float* out,
                 cudaStream_t st);
// One pass from the logits: logp, the policy loss and, where dz is given, the
// logits' gradient times grad_scale.
int policy_loss_logits(const LogitRows& r, const Packed& p, const PolicyTerms& t, float grad_scale,
                       float* values, float* logp, void* dz, int64_t dz_stride, void* ws,
                       size_t ws_bytes, cudaStream_t st);
size_t policy_logits_workspace_bytes(int64_t rows, int64_t count);
// rows of dz times g[0] / grad_scale, in place; nothing where that is 1.
int scale_rows(void* dz, int dtype, int64_t stride, int64_t rows, int64_t vocab, const float* g,
               float grad_scale, cudaStream_t st);

}  // namespace sinkslot
