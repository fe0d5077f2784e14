// Internal interface between the C ABI of sampling (dz_prefix_api.hip) and its
// kernel (dz_sampling.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dz {

struct SampleRows {
  const void* logits;
  int64_t stride;
  uint32_t nrows, vocab;
  const float* uniform;
  // one for each row, or (NULL) the same for all
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  double temperature, top_p, min_p;
  int32_t top_k;
  int64_t* tokens;
};
constexpr uint32_t kMaxSampleVocab = 1u << 20;

hipError_t launch_sample(int dtype, const SampleRows& a, hipStream_t st);

}  // namespace dz
