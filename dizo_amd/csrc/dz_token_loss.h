// Internal interface between the C ABI of the vocabulary operators
// (dz_token_api.hip) and their kernels (dz_token_loss.hip, dz_token_head.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dz_common.h"

namespace dz {

// `batch` x `length` rows of a tensor, by element strides.
struct RowStrides {
  int64_t batch, row;
};

// Rows of logits and what is read from and written for each. Row r is
// sequence r / length, position r % length; outputs without strides are dense.
struct VocabRows {
  const void* logits;
  RowStrides logits_s;
  uint32_t nrows, length, vocab;
  // token_logprobs
  const int64_t* tokens;
  RowStrides tokens_s;
  int64_t ignore;
  int32_t top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  const float* entropy_weights;  // may be NULL: no entropy term in the gradient
  RowStrides entropy_weights_s;
  // topk_distill
  const float* teacher_values;    // (nrows, k)
  const int64_t* teacher_tokens;  // (nrows, k), -1: no entry
  int32_t k;
  int32_t normalize;
  float temperature;
  float* loss;
  // gradient (grad != NULL)
  const float* weights;  // token_logprobs: may be NULL (zeros)
  RowStrides weights_s;
  void* grad;
  RowStrides grad_s;
  bool past_caches;  // of the gradient's stores
};

constexpr int kMaxTop = 128;      // alternatives of a row
constexpr int kMaxTeacher = 512;  // a teacher's entries of a row

hipError_t launch_token_logprobs(int dtype, const VocabRows& a, hipStream_t st);
hipError_t launch_topk_distill(int dtype, const VocabRows& a, hipStream_t st);

// Log probabilities straight from hidden states and the head.
struct HeadRows {
  const void* hidden;  // (nrows, width), rows hidden_stride apart
  const void* weight;  // (vocab, width), rows weight_stride apart
  int64_t hidden_stride, weight_stride;
  uint32_t nrows, width, vocab;
  const int64_t* tokens;
  int64_t ignore;
  float* logprobs;
  float* entropy;
};
// Bytes of the workspace of a launch, whatever the tokens are.
int64_t head_workspace(int dtype, uint32_t nrows, uint32_t width, uint32_t vocab);
hipError_t launch_head(int dtype, const HeadRows& a, void* workspace, hipStream_t st);

}  // namespace dz
