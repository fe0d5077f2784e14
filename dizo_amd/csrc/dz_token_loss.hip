// Kernels over rows of logits: log probabilities of given tokens with the
// rows' entropies and largest alternatives, the distance to a teacher's
// largest logits, and their gradients.
#include "dz_token_loss.h"
#include "dz_token_math.h"

namespace dz {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct Shared {
  SoftStats wave[kWaves];
  uint64_t best[kWaves];
  float w[kMaxTeacher], lnw[kMaxTeacher];
  int32_t idx[kMaxTeacher];
  float red[kWaves];
};

__device__ SoftStats block_stats(SoftStats st, float c, Shared& sh) {
  for (int off = 32; off >= 1; off >>= 1) {
    SoftStats o;
    o.m = __shfl_xor(st.m, off, 64);
    o.s = __shfl_xor(st.s, off, 64);
    o.t = __shfl_xor(st.t, off, 64);
    st.join(o, c);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = st;
  __syncthreads();
  st = sh.wave[0];
  for (int i = 1; i < kWaves; ++i) st.join(sh.wave[i], c);
  return st;
}

template <bool MAX>
__device__ float block_reduce(float v, Shared& sh) {
  for (int off = 32; off >= 1; off >>= 1) {
    const float o = __shfl_xor(v, off, 64);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.red[0];
  for (int i = 1; i < kWaves; ++i) v = MAX ? fmaxf(v, sh.red[i]) : v + sh.red[i];
  return v;
}

// Orders (logit, index): larger logits first, equal ones by index. Keys of
// different indexes differ; 0 is below every key. -0 and +0 are equal.
__device__ uint64_t order_key(float x, uint32_t i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~i;
}
__device__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

template <class T>
__device__ SoftStats row_stats(const typename T::Elem* x, uint32_t v, float c, Shared& sh) {
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < v; i += kThreads) m = fmaxf(m, T::load(x + i));
  SoftStats st = SoftStats::of(m);
  for (uint32_t i = threadIdx.x; i < v; i += kThreads) st.add(T::load(x + i), c);
  return block_stats(st, c, sh);
}

template <class T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(VocabRows a) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x, b = r / a.length, l = r % a.length, tid = threadIdx.x;
  const typename T::Elem* x = (const typename T::Elem*)a.logits + b * a.logits_s.batch + l * a.logits_s.row;
  typename T::Elem* g = a.grad ? (typename T::Elem*)a.grad + b * a.grad_s.batch + l * a.grad_s.row : nullptr;
  const int64_t tok = a.tokens[b * a.tokens_s.batch + l * a.tokens_s.row];
  if (tok == a.ignore) {
    if (tid == 0) {
      a.logprobs[r] = 0.f;
      a.entropy[r] = 0.f;
    }
    for (int i = tid; i < a.top; i += kThreads) {
      a.top_logprobs[(int64_t)r * a.top + i] = -INFINITY;
      a.top_tokens[(int64_t)r * a.top + i] = -1;
    }
    if (g)
      for (uint32_t i = tid; i < a.vocab; i += kThreads) T::store(g + i, 0.f);
    return;
  }
  const SoftStats st = row_stats<T>(x, a.vocab, kLog2e, sh);
  const bool valid = st.valid();
  const float log2s = log2_hw(st.s);
  const float entropy = valid ? kLn2 * (log2s - st.t / st.s) : NAN;
  const bool inside = tok >= 0 && tok < (int64_t)a.vocab;
  if (tid == 0) {
    a.logprobs[r] = valid && inside ? st.lnq(T::load(x + tok), 1.f) : NAN;
    a.entropy[r] = entropy;
  }
  uint64_t prev = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    uint64_t best = 0;
    if (valid)
      for (uint32_t i = tid; i < a.vocab; i += kThreads) {
        const uint64_t k = order_key(T::load(x + i), i);
        if (k < prev && k > best) best = k;
      }
    for (int off = 32; off >= 1; off >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, off, 64);
      best = o > best ? o : best;
    }
    __syncthreads();
    if ((tid & 63) == 0) sh.best[tid >> 6] = best;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) best = sh.best[i] > best ? sh.best[i] : best;
    prev = best;
    if (tid == 0) {
      a.top_logprobs[(int64_t)r * a.top + j] = valid ? st.lnq(key_value(best), 1.f) : NAN;
      a.top_tokens[(int64_t)r * a.top + j] = valid ? (int64_t)(uint32_t)~(uint32_t)best : -1;
    }
  }
  if (!g) return;
  const float w = a.weights ? a.weights[b * a.weights_s.batch + l * a.weights_s.row] : 0.f;
  const float u = a.entropy_weights ? a.entropy_weights[b * a.entropy_weights_s.batch + l * a.entropy_weights_s.row] : 0.f;
  for (uint32_t i = tid; i < a.vocab; i += kThreads) {
    const float z = st.y_of(T::load(x + i), kLog2e) - log2s;  // log2 q
    const float q = exp2_hw(z);
    float d = -q * (w + u * __builtin_fmaf(kLn2, fmaxf(z, -1e30f), entropy));
    if ((int64_t)i == tok) d += w;
    T::store(g + i, valid && inside ? d : NAN);
  }
}

template <class T>
__global__ __launch_bounds__(kThreads) void topk_distill_kernel(VocabRows a) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x, b = r / a.length, l = r % a.length, tid = threadIdx.x;
  const typename T::Elem* x = (const typename T::Elem*)a.logits + b * a.logits_s.batch + l * a.logits_s.row;
  typename T::Elem* g = a.grad ? (typename T::Elem*)a.grad + b * a.grad_s.batch + l * a.grad_s.row : nullptr;
  // the teacher's softmax over its entries; one outside the vocabulary makes the row NaN
  float tm = -INFINITY;
  int any = 0, bad = 0;
  for (int j = tid; j < a.k; j += kThreads) {
    const int64_t i = a.teacher_tokens[(int64_t)r * a.k + j];
    const bool in = i >= 0 && i < (int64_t)a.vocab;
    const float t = a.teacher_values[(int64_t)r * a.k + j] / (a.normalize ? a.temperature : 1.f);
    any |= i != -1;
    bad |= i != -1 && (!in || !(t < INFINITY));
    sh.idx[j] = in ? (int32_t)i : -1;
    sh.lnw[j] = in ? t : -INFINITY;
    if (in) tm = fmaxf(tm, t);
  }
  any = __syncthreads_or(any);
  bad = __syncthreads_or(bad);
  if (!any) {
    if (tid == 0) a.loss[r] = 0.f;
    if (g)
      for (uint32_t i = tid; i < a.vocab; i += kThreads) T::store(g + i, 0.f);
    return;
  }
  float lse = 0.f;
  if (a.normalize) {
    tm = block_reduce<true>(tm, sh);
    float s = 0.f;
    for (int j = tid; j < a.k; j += kThreads)
      if (sh.idx[j] >= 0) s += exp2_hw((sh.lnw[j] - tm) * kLog2e);
    s = block_reduce<false>(s, sh);
    lse = tm + kLn2 * log2_hw(s);
    bad |= tm == -INFINITY;
  }
  float total = 0.f;
  for (int j = tid; j < a.k; j += kThreads) {
    const float lnw = sh.lnw[j] - lse;
    const float w = sh.idx[j] >= 0 ? exp2_hw(lnw * kLog2e) : 0.f;
    sh.lnw[j] = lnw;
    sh.w[j] = w;
    total += w;
  }
  total = block_reduce<false>(total, sh);

  const float c = kLog2e / a.temperature;
  const SoftStats st = row_stats<T>(x, a.vocab, c, sh);
  const float log2s = log2_hw(st.s);
  bad |= !st.valid();
  float loss = 0.f;
  for (int j = tid; j < a.k; j += kThreads)
    if (sh.w[j] > 0.f) loss += sh.w[j] * (sh.lnw[j] - st.lnq(T::load(x + sh.idx[j]), 1.f / a.temperature));
  loss = block_reduce<false>(loss, sh);
  const float tau = a.temperature;
  if (tid == 0) a.loss[r] = bad ? NAN : tau * tau * loss;
  if (!g) return;
  const float up = bad ? NAN : tau * a.weights[b * a.weights_s.batch + l * a.weights_s.row];
  for (uint32_t i = tid; i < a.vocab; i += kThreads)
    T::store(g + i, up * (total * exp2_hw(st.y_of(T::load(x + i), c) - log2s)));
  __syncthreads();
  // the teacher's entries, each written by the first that names its token
  for (int j = tid; j < a.k; j += kThreads) {
    const int32_t i = sh.idx[j];
    if (i < 0) continue;
    bool first = true;
    float w = 0.f;
    for (int h = 0; h < a.k; ++h)
      if (sh.idx[h] == i) {
        if (h < j) first = false;
        w += sh.w[h];
      }
    if (first) T::store(g + i, up * (total * exp2_hw(st.y_of(T::load(x + i), c) - log2s) - w));
  }
}

}  // namespace

#define DZ_BY_TYPE(KERNEL, grid, st, args)                                        \
  do {                                                                            \
    if (dtype == DZ_F32) KERNEL<TypeF32><<<grid, kThreads, 0, st>>>(args);        \
    else if (dtype == DZ_F16) KERNEL<TypeF16><<<grid, kThreads, 0, st>>>(args);   \
    else KERNEL<TypeBF16><<<grid, kThreads, 0, st>>>(args);                       \
  } while (0)

hipError_t launch_token_logprobs(int dtype, const VocabRows& a, hipStream_t st) {
  DZ_BY_TYPE(token_logprobs_kernel, a.nrows, st, a);
  return hipGetLastError();
}

hipError_t launch_topk_distill(int dtype, const VocabRows& a, hipStream_t st) {
  DZ_BY_TYPE(topk_distill_kernel, a.nrows, st, a);
  return hipGetLastError();
}

}  // namespace dz
