// Device helpers of the vocabulary operators: elements of the three types as
// fp32, and softmax statistics that can be joined.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dz_common.h"

namespace dz {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// An element type, and 16 bytes of it.
struct TypeF32 {
  using Elem = float;
  using V = f32x4;
  static constexpr int kPer16 = 4;
};
struct TypeF16 {
  using Elem = _Float16;
  using V = f16x8;
  static constexpr int kPer16 = 8;
};
struct TypeBF16 {
  using Elem = __bf16;
  using V = bf16x8;
  static constexpr int kPer16 = 8;
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

// Statistics of logits x: their maximum m, s = sum 2^y and t = sum 2^y y with
// y = (x - m) c (c = log2 e / temperature). Then log softmax(x) = (x - m) / temperature -
// ln 2 log2 s and the entropy is ln 2 (log2 s - t / s): both of its terms are of one sign.
struct SoftStats {
  float m, s, t;

  __device__ static SoftStats of(float m) { return SoftStats{m, 0.f, 0.f}; }

  // y of one logit; no logits above -inf: y of any is taken against 0, so that 2^y is 0
  __device__ float y_of(float x, float c) const { return (x - (m == -INFINITY ? 0.f : m)) * c; }

  // log softmax of one logit, with `inv` the inverse of the temperature. Not from y:
  // a logit near the type's lowest value has a y past the range of fp32.
  __device__ float lnq(float x, float inv) const { return __builtin_fmaf(-kLn2, log2_hw(s), (x - m) * inv); }

  // 2^y y is 0 where y is -inf; a NaN logit leaves a NaN in s
  template <bool ENTROPY = true>
  __device__ void add(float x, float c) {
    const float y = y_of(x, c);
    const float e = exp2_hw(y);
    s += e;
    if (ENTROPY) t = __builtin_fmaf(e, fmaxf(y, -1e30f), t);
  }

  // The same statistics against another maximum, m2 >= m.
  __device__ void rebase(float m2, float c) {
    if (s != 0.f) {  // a NaN passes
      const float d = (m - m2) * c;
      const float f = exp2_hw(d);
      t = f * __builtin_fmaf(fmaxf(d, -1e30f), s, t);
      s *= f;
    }
    m = m2;
  }
  __device__ void join(SoftStats o, float c) {
    const float m2 = fmaxf(m, o.m);
    rebase(m2, c);
    o.rebase(m2, c);
    s += o.s;
    t += o.t;
  }
  // A distribution: at least one finite logit, and no NaN or +inf.
  __device__ bool valid() const { return s == s && fabsf(m) != INFINITY; }
};

}  // namespace dz
