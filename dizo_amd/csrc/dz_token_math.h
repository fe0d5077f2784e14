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
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
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

// 2^y is 0 from y = -150 on; a product with y takes no less than this for it, so that it is 0 there too
// (-inf would make it a NaN, and a large bound one that overflows with a factor beside it).
constexpr float kLowestY = -256.f;

// Statistics of logits x: their maximum m, s = sum 2^y and t = sum 2^y y with y = x c - K,
// c = log2 e / temperature. K is m c rounded to fp32: what its rounding leaves shifts every y alike,
// so that log softmax(x) = ln 2 (y - log2 s) and the entropy ln 2 (log2 s - t / s), of which both terms
// are of one sign, do not see it, and y is one fused multiply-add. Where m c leaves the range of
// fp32 (logits at the type's limits), and where no logit is above -inf, y = (x - m) c instead; FAR
// takes that everywhere: y is 0 for the largest logit, and so are the gradients of a row that
// is certain.
template <bool FAR>
struct Stats {
  float m, s, t;

  __device__ static Stats of(float m) { return Stats{m, 0.f, 0.f}; }

  __device__ static bool in_range(float k) { return !FAR && fabsf(k) < 1e37f; }
  __device__ bool plain(float c) const { return in_range(m * c); }
  __device__ float y_plain(float x, float c) const { return __builtin_fmaf(x, c, -(m * c)); }
  // no logits above -inf: y of any is taken against 0, so that 2^y is 0
  __device__ float y_far(float x, float c) const { return (x - (m == -INFINITY ? 0.f : m)) * c; }
  __device__ float y_of(float x, float c) const { return plain(c) ? y_plain(x, c) : y_far(x, c); }

  // log softmax of one logit, with `inv` the inverse of the temperature. A logit near the
  // type's lowest value has a y past the range of fp32.
  __device__ float lnq(float x, float c, float inv) const {
    const float y = y_of(x, c);
    return y == -INFINITY ? __builtin_fmaf(-kLn2, log2_hw(s), (x - m) * inv) : kLn2 * (y - log2_hw(s));
  }

  // Adds x(0) .. x(N - 1). (A NaN logit leaves a NaN in s.)
  template <bool ENTROPY, int N, class F>
  __device__ __forceinline__ void add_far(F x, float c) {
    const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float y = (x(i) - m0) * c;
      if (!FAR) y = in_range(m * c) ? y_plain(x(i), c) : y;
      const float e = exp2_hw(y);
      s += e;
      if (ENTROPY) t = __builtin_fmaf(e, fmaxf(y, kLowestY), t);
    }
  }
  // The same with one operation for y, and none for its limit unless it is met.
  template <bool ENTROPY, int N, class F>
  __device__ __forceinline__ void add(F x, float c) {
    const float k = m * c, s0 = s, t0 = t;
    if (__all(in_range(k))) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float y = __builtin_fmaf(x(i), c, -k);
        const float e = exp2_hw(y);
        s += e;
        if (ENTROPY) t = __builtin_fmaf(e, y, t);
      }
      if (!ENTROPY || !__any(t != t)) return;
      s = s0;
      t = t0;
    }
    asm("" : "+v"(c));  // or the compiler keeps all of the first pass's values for this one
    add_far<ENTROPY, N>(x, c);
  }

  // The same statistics against another maximum, m2 >= m.
  __device__ void rebase(float m2, float c) {
    if (s != 0.f) {  // a NaN passes
      const float k = m * c, k2 = m2 * c;
      const float d = in_range(k) && in_range(k2) ? k - k2 : (m - m2) * c;
      const float f = exp2_hw(d);
      t = f * __builtin_fmaf(fmaxf(d, kLowestY), s, t);
      s *= f;
    }
    m = m2;
  }
  __device__ void join(Stats o, float c) {
    const float m2 = fmaxf(m, o.m);
    rebase(m2, c);
    o.rebase(m2, c);
    s += o.s;
    t += o.t;
  }
  // A distribution: at least one finite logit, and no NaN or +inf.
  __device__ bool valid() const { return s == s && fabsf(m) != INFINITY; }
};
using SoftStats = Stats<false>;

}  // namespace dz
