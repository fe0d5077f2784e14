// C ABI of the vocabulary operators (declared in include/dizo_amd.h):
// argument checks, then one launch each (linear_token_logprobs: three).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "../../include/dizo_amd.h"
#include "dz_common.h"
#include "dz_internal.h"
#include "dz_token_loss.h"

namespace {

using dz::api_fail;

// A launch's grid is rows x 1,024 threads at most, and counts threads in 32 bits.
constexpr int64_t kMaxRows = (1 << 22) - 1;
// Row indexes and vector counts stay in 32 bits.
constexpr int64_t kMaxVocab = (int64_t)1 << 30;

int32_t check_common(int32_t dtype, int64_t batch, int64_t length, int64_t vocab) {
  if (dtype != DZ_DTYPE_F32 && dtype != DZ_DTYPE_F16 && dtype != DZ_DTYPE_BF16)
    return api_fail(DZ_ERR_INVALID, "unknown dtype code " + std::to_string(dtype));
  if (batch < 0 || length < 0 || (batch > 0 && length > kMaxRows / batch))
    return api_fail(DZ_ERR_INVALID, "row count out of range: " + std::to_string(batch) + " x " + std::to_string(length) +
                                        " (at most " + std::to_string(kMaxRows) + " rows)");
  if (vocab < 1 || vocab > kMaxVocab)
    return api_fail(DZ_ERR_INVALID, "vocab out of range: " + std::to_string(vocab));
  return DZ_OK;
}

// A strided operand: strides not negative, and its extent inside one allocation.
// (`rows` of `inner` elements each.)
int32_t check_strided(const void* p, int64_t es, int64_t batch, int64_t length, int64_t bs, int64_t ls, int64_t inner,
                      const char* what) {
  if (!p) return api_fail(DZ_ERR_INVALID, std::string(what) + " is NULL");
  if (bs < 0 || ls < 0) return api_fail(DZ_ERR_INVALID, std::string(what) + ": negative stride");
  constexpr int64_t kMost = (int64_t)1 << 52;
  if (bs > kMost / batch || ls > kMost / length) return api_fail(DZ_ERR_INVALID, std::string(what) + ": stride out of range");
  const int64_t extent = (batch - 1) * bs + (length - 1) * ls + inner;
  if ((uintptr_t)p % (uintptr_t)es) return api_fail(DZ_ERR_INVALID, std::string(what) + " is not aligned to its elements");
  return dz::api_check_range(p, (uint64_t)extent * (uint64_t)es, what);
}

int32_t check_dense(const void* p, int64_t es, int64_t n, const char* what) {
  return check_strided(p, es, 1, 1, 0, 0, n, what);
}

// Rows that are written must not share elements.
int32_t check_distinct(int64_t batch, int64_t length, int64_t bs, int64_t ls, int64_t inner, const char* what) {
  const bool rows_apart = length == 1 || ls >= inner;
  const bool batches_apart = batch == 1 || bs >= (length - 1) * ls + inner ||
                             (length > 1 && bs >= inner && ls >= (batch - 1) * bs + inner);
  if (!rows_apart || !batches_apart) return api_fail(DZ_ERR_INVALID, std::string(what) + ": rows overlap");
  return DZ_OK;
}

// A gradient may be written over its logits, row over row; otherwise the ranges from first to last element lie apart.
int32_t check_apart(const void* logits, const void* grad, int64_t es, int64_t batch, int64_t length, int64_t vocab, int64_t logits_bs,
                    int64_t logits_ls, int64_t grad_bs, int64_t grad_ls) {
  if (logits == grad && (batch == 1 || logits_bs == grad_bs) && (length == 1 || logits_ls == grad_ls)) return DZ_OK;
  const uint64_t x = (uint64_t)(uintptr_t)logits, g = (uint64_t)(uintptr_t)grad;
  const uint64_t x_end = x + (uint64_t)(((batch - 1) * logits_bs + (length - 1) * logits_ls + vocab) * es);
  const uint64_t g_end = g + (uint64_t)(((batch - 1) * grad_bs + (length - 1) * grad_ls + vocab) * es);
  if (x < g_end && g < x_end) return api_fail(DZ_ERR_INVALID, "grad and logits overlap");
  return DZ_OK;
}

int64_t size_of(int32_t dtype) { return dtype == DZ_DTYPE_F32 ? 4 : 2; }

int32_t launched(hipError_t e, const char* what) { return e == hipSuccess ? DZ_OK : dz::api_hip_fail(e, what); }

}  // namespace

#define DZ_TRY(expr)             \
  do {                           \
    const int32_t rc_ = (expr);  \
    if (rc_) return rc_;         \
  } while (0)

extern "C" {

int32_t dz_token_logprobs(const void* logits, int32_t dtype, int64_t batch, int64_t length, int64_t vocab,
                          int64_t logits_bs, int64_t logits_ls, const int64_t* tokens, int64_t tokens_bs,
                          int64_t tokens_ls, int64_t ignore_index, int32_t top, float* logprobs, float* entropy,
                          float* top_logprobs, int64_t* top_tokens, const float* weights, int64_t weights_bs,
                          int64_t weights_ls, const float* entropy_weights, int64_t entropy_weights_bs,
                          int64_t entropy_weights_ls, void* grad, int64_t grad_bs, int64_t grad_ls, void* stream) {
  DZ_TRY(check_common(dtype, batch, length, vocab));
  if (top < 0 || top > dz::kMaxTop || top > vocab)
    return api_fail(DZ_ERR_INVALID, "top out of range: " + std::to_string(top) + " of " + std::to_string(vocab) +
                                        " tokens (at most " + std::to_string(dz::kMaxTop) + ")");
  if (top && grad) return api_fail(DZ_ERR_INVALID, "top and grad exclude each other");
  if (batch * length == 0) return DZ_OK;
  const int64_t es = size_of(dtype), n = batch * length;
  DZ_TRY(check_strided(logits, es, batch, length, logits_bs, logits_ls, vocab, "logits"));
  DZ_TRY(check_strided(tokens, 8, batch, length, tokens_bs, tokens_ls, 1, "tokens"));
  DZ_TRY(check_dense(logprobs, 4, n, "logprobs"));
  DZ_TRY(check_dense(entropy, 4, n, "entropy"));
  if (top) {
    DZ_TRY(check_dense(top_logprobs, 4, n * top, "top_logprobs"));
    DZ_TRY(check_dense(top_tokens, 8, n * top, "top_tokens"));
  }
  if (grad) {
    if (!weights && !entropy_weights) return api_fail(DZ_ERR_INVALID, "a gradient needs weights or entropy_weights");
    DZ_TRY(check_strided(grad, es, batch, length, grad_bs, grad_ls, vocab, "grad"));
    DZ_TRY(check_distinct(batch, length, grad_bs, grad_ls, vocab, "grad"));
    DZ_TRY(check_apart(logits, grad, es, batch, length, vocab, logits_bs, logits_ls, grad_bs, grad_ls));
    if (weights) DZ_TRY(check_strided(weights, 4, batch, length, weights_bs, weights_ls, 1, "weights"));
    if (entropy_weights)
      DZ_TRY(check_strided(entropy_weights, 4, batch, length, entropy_weights_bs, entropy_weights_ls, 1, "entropy_weights"));
  }
  dz::VocabRows a{};
  a.logits = logits;
  a.logits_s = {logits_bs, logits_ls};
  a.nrows = (uint32_t)n;
  a.length = (uint32_t)length;
  a.vocab = (uint32_t)vocab;
  a.tokens = tokens;
  a.tokens_s = {tokens_bs, tokens_ls};
  a.ignore = ignore_index;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_tokens = top_tokens;
  a.weights = weights;
  a.weights_s = {weights_bs, weights_ls};
  a.entropy_weights = entropy_weights;
  a.entropy_weights_s = {entropy_weights_bs, entropy_weights_ls};
  a.grad = grad;
  a.grad_s = {grad_bs, grad_ls};
  return launched(dz::launch_token_logprobs(dtype, a, (hipStream_t)stream), "token_logprobs kernel launch");
}

int32_t dz_topk_distill(const void* logits, int32_t dtype, int64_t batch, int64_t length, int64_t vocab,
                        int64_t logits_bs, int64_t logits_ls, const float* teacher_values,
                        const int64_t* teacher_tokens, int32_t k, float temperature, int32_t normalize, float* loss,
                        const float* weights, int64_t weights_bs, int64_t weights_ls, void* grad, int64_t grad_bs,
                        int64_t grad_ls, void* stream) {
  DZ_TRY(check_common(dtype, batch, length, vocab));
  if (k < 1 || k > dz::kMaxTeacher)
    return api_fail(DZ_ERR_INVALID, "teacher entries out of range: " + std::to_string(k) + " (1 to " +
                                        std::to_string(dz::kMaxTeacher) + ")");
  // the loss has the square as a factor: one that is 0 or infinite leaves nothing of it, and the inverse
  // times log2 e is finite then
  if (!(temperature > 0.f) || !isnormal(temperature * temperature))
    return api_fail(DZ_ERR_INVALID, "temperature must be positive and finite, and so its square (2^-63 to 2^64)");
  if (batch * length == 0) return DZ_OK;
  const int64_t es = size_of(dtype), n = batch * length;
  DZ_TRY(check_strided(logits, es, batch, length, logits_bs, logits_ls, vocab, "logits"));
  DZ_TRY(check_dense(teacher_values, 4, n * k, "teacher_values"));
  DZ_TRY(check_dense(teacher_tokens, 8, n * k, "teacher_tokens"));
  DZ_TRY(check_dense(loss, 4, n, "loss"));
  if (grad) {
    DZ_TRY(check_strided(grad, es, batch, length, grad_bs, grad_ls, vocab, "grad"));
    DZ_TRY(check_distinct(batch, length, grad_bs, grad_ls, vocab, "grad"));
    DZ_TRY(check_apart(logits, grad, es, batch, length, vocab, logits_bs, logits_ls, grad_bs, grad_ls));
    DZ_TRY(check_strided(weights, 4, batch, length, weights_bs, weights_ls, 1, "weights"));
  }
  dz::VocabRows a{};
  a.logits = logits;
  a.logits_s = {logits_bs, logits_ls};
  a.nrows = (uint32_t)n;
  a.length = (uint32_t)length;
  a.vocab = (uint32_t)vocab;
  a.teacher_values = teacher_values;
  a.teacher_tokens = teacher_tokens;
  a.k = k;
  a.normalize = normalize != 0;
  a.temperature = temperature;
  a.loss = loss;
  a.weights = weights;
  a.weights_s = {weights_bs, weights_ls};
  a.grad = grad;
  a.grad_s = {grad_bs, grad_ls};
  return launched(dz::launch_topk_distill(dtype, a, (hipStream_t)stream), "topk_distill kernel launch");
}

int32_t dz_linear_token_logprobs_workspace(int32_t dtype, int64_t rows, int64_t width, int64_t vocab, int64_t* bytes) {
  DZ_TRY(check_common(dtype, rows, 1, vocab));
  if (width < 1 || width > kMaxVocab) return api_fail(DZ_ERR_INVALID, "width out of range: " + std::to_string(width));
  if (!bytes) return api_fail(DZ_ERR_INVALID, "bytes is NULL");
  *bytes = rows ? dz::head_workspace(dtype, (uint32_t)rows, (uint32_t)width, (uint32_t)vocab) : 0;
  return DZ_OK;
}

int32_t dz_linear_token_logprobs(const void* hidden, const void* weight, int32_t dtype, int64_t rows, int64_t width,
                                 int64_t vocab, int64_t hidden_stride, int64_t weight_stride, const int64_t* tokens,
                                 int64_t ignore_index, float* logprobs, float* entropy, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  DZ_TRY(dz_linear_token_logprobs_workspace(dtype, rows, width, vocab, &need));
  if (rows == 0) return DZ_OK;
  const int64_t es = size_of(dtype);
  DZ_TRY(check_strided(hidden, es, 1, rows, 0, hidden_stride, width, "hidden"));
  DZ_TRY(check_strided(weight, es, 1, vocab, 0, weight_stride, width, "weight"));
  DZ_TRY(check_dense(tokens, 8, rows, "tokens"));
  DZ_TRY(check_dense(logprobs, 4, rows, "logprobs"));
  DZ_TRY(check_dense(entropy, 4, rows, "entropy"));
  if (workspace_bytes < need)
    return api_fail(DZ_ERR_INVALID, "workspace of " + std::to_string(workspace_bytes) + " bytes: " + std::to_string(need) + " are needed");
  DZ_TRY(check_dense(workspace, 16, (need + 15) / 16, "workspace"));
  dz::HeadRows a{};
  a.hidden = hidden;
  a.weight = weight;
  a.hidden_stride = hidden_stride;
  a.weight_stride = weight_stride;
  a.nrows = (uint32_t)rows;
  a.width = (uint32_t)width;
  a.vocab = (uint32_t)vocab;
  a.tokens = tokens;
  a.ignore = ignore_index;
  a.logprobs = logprobs;
  a.entropy = entropy;
  return launched(dz::launch_head(dtype, a, workspace, (hipStream_t)stream), "linear_token_logprobs kernel launch");
}

}  // extern "C"
