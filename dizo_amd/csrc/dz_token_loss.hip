// Kernels over rows of logits: log probabilities of given tokens with the
// rows' entropies and largest alternatives, the distance to a teacher's
// largest logits, and their gradients.
//
// One workgroup takes one row. What bounds these kernels is reading the row
// once (and writing its gradient once), so a row that fits is held in the
// workgroup's registers as it was read, in 16-byte vectors: the statistics, the
// alternatives and the gradient are all taken from there. A longer row goes by
// in chunks of as much, and is read again for the later passes. A thread's
// vectors lie THREADS apart, so that a wave's loads cover consecutive bytes.
//
// Rows start where they start (an odd vocabulary, a view): vectors are taken at
// the 16-byte boundaries of memory, and the row's first and last one, where they
// are not whole, element by element, so that nothing outside the row is read.
#include "dz_token_loss.h"
#include "dz_token_math.h"

#include <type_traits>

namespace dz {
namespace {

constexpr uint32_t kCandidates = 2048;  // alternatives that a row's threshold may leave over
constexpr uint32_t kGroups = 256;       // of threads, whose maxima give the threshold

// ------------------------------------------------------------- reductions --
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
// Over 16 lanes: lanes 1, then 2 apart within fours, then mirrored within eights and sixteens.
template <class F>
__device__ __forceinline__ float reduce16(float x, F f) {
  x = f(x, dpp<0xB1>(x));
  x = f(x, dpp<0x4E>(x));
  x = f(x, dpp<0x141>(x));
  return f(x, dpp<0x140>(x));
}
template <class F>
__device__ __forceinline__ float reduce64(float x, F f) {
  x = reduce16(x, f);
  x = f(x, __shfl_xor(x, 16, 64));
  return f(x, __shfl_xor(x, 32, 64));
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
  __device__ float operator()(float a, float b) const { return a + b; }
};

template <int THREADS, bool ENTROPY, bool FAR>
__device__ __forceinline__ Stats<FAR> block_stats(Stats<FAR> st, float c, Stats<FAR>* waves) {
  constexpr uint32_t W = THREADS / 64;
  const uint32_t lane = threadIdx.x & 63;
  st.rebase(reduce64(st.m, Max()), c);
  st.s = reduce64(st.s, Add());
  if (ENTROPY) st.t = reduce64(st.t, Add());
  if (lane == 0) waves[threadIdx.x >> 6] = st;
  __syncthreads();
  st = waves[lane < W ? lane : 0];
  if (lane >= W) st = Stats<FAR>::of(-INFINITY);
  st.rebase(reduce16(st.m, Max()), c);  // W <= 16: lanes 0 .. 15 hold them all
  st.s = reduce16(st.s, Add());
  if (ENTROPY) st.t = reduce16(st.t, Add());
  st.m = __shfl(st.m, 0, 64);
  st.s = __shfl(st.s, 0, 64);
  st.t = __shfl(st.t, 0, 64);
  return st;
}

// --------------------------------------------------------------- the row --
// The 16-byte vectors that v elements at p lie in.
template <class T>
struct Span {
  using Elem = typename T::Elem;
  static constexpr uint32_t E = T::kPer16;
  uint64_t base;      // of vector 0
  uint32_t lead;      // elements of vector 0 before the row
  uint32_t v;
  uint32_t nvec;      // vectors
  uint32_t end_full;  // vector end_full is the last one where it is not whole

  __device__ Span(const void* p, uint32_t n) {
    const uint64_t a = (uint64_t)p;
    base = a & ~(uint64_t)15;
    lead = (uint32_t)(a & 15) / sizeof(Elem);
    v = n;
    end_full = (v + lead) / E;
    nvec = (v + lead + E - 1) / E;
  }
  __device__ bool whole(uint32_t j) const { return j >= (lead ? 1u : 0u) && j < end_full; }
  __device__ uint32_t first(uint32_t j) const { return j * E - lead; }  // index of a vector's element 0 (wraps below 0)
  __device__ const Elem* row() const { return (const Elem*)base + lead; }

  __device__ u32x4 edge(uint32_t j) const {
    typename T::V x;
    for (uint32_t k = 0; k < E; ++k) {
      const uint32_t i = first(j) + k;
      x[k] = i < v ? row()[i] : (Elem)-INFINITY;
    }
    return __builtin_bit_cast(u32x4, x);
  }
};

template <class T>
__device__ __forceinline__ u32x4 none16() {  // no logits: -inf
  typename T::V x;
  for (int k = 0; k < T::kPer16; ++k) x[k] = (typename T::Elem)-INFINITY;
  return __builtin_bit_cast(u32x4, x);
}
template <class T>
__device__ __forceinline__ float element(const u32x4& raw, int k) {
  return (float)__builtin_bit_cast(typename T::V, raw)[k];
}

// THREADS x NV vectors of a row from vector j0 on, in registers.
template <class T, int THREADS, int NV>
struct Held {
  u32x4 raw[NV];

  __device__ __forceinline__ static uint32_t index(uint32_t j0, int i) { return j0 + i * THREADS + threadIdx.x; }

  __device__ __forceinline__ void load(const Span<T>& s, uint32_t j0) {
    const uint32_t tail = s.end_full < s.nvec ? s.end_full : ~0u;
    u32x4 last = none16<T>();
    if (tail != ~0u && tail % THREADS == threadIdx.x) last = s.edge(tail);  // j0 is a multiple of THREADS
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t j = index(j0, i);
      raw[i] = none16<T>();
      if (s.whole(j)) raw[i] = *(const u32x4*)(s.base + (uint64_t)j * 16);
      if (j == tail) raw[i] = last;
    }
    if (s.lead && tail != 0 && index(j0, 0) == 0) raw[0] = s.edge(0);
  }
  __device__ __forceinline__ float largest() const {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < T::kPer16; ++k) m = fmaxf(m, element<T>(raw[i], k));
    return m;
  }
  template <bool ENTROPY, bool FAR>
  __device__ __forceinline__ void add_to(Stats<FAR>& st, float c) const {
    st.template add<ENTROPY, NV * T::kPer16>([&](int i) { return element<T>(raw[i / T::kPer16], i % T::kPer16); }, c);
  }
};

// A row's softmax statistics. Leaves the row in `h` where it fits.
template <class T, int THREADS, int NV, bool ENTROPY, bool FAR>
__device__ __forceinline__ Stats<FAR> row_stats(const Span<T>& s, Held<T, THREADS, NV>& h, float c, Stats<FAR>* waves) {
  auto st = Stats<FAR>::of(-INFINITY);
  for (uint32_t j0 = 0; j0 < s.nvec; j0 += THREADS * NV) {
    h.load(s, j0);
    st.rebase(fmaxf(st.m, h.largest()), c);
    h.template add_to<ENTROPY>(st, c);
  }
  return block_stats<THREADS, ENTROPY>(st, c, waves);
}

// Writes f(logit, index) for the whole row. Vector by vector where the output
// lies at the input's place within 16 bytes, else element by element.
template <class T, int THREADS, int NV, class F>
__device__ __forceinline__ void write_row(const Span<T>& s, Held<T, THREADS, NV>& h, typename T::Elem* out, F f) {
  const Span<T> o(out, s.v);
  if (o.lead != s.lead) {
    const typename T::Elem* x = s.row();
    for (uint32_t i = threadIdx.x; i < s.v; i += THREADS) out[i] = (typename T::Elem)f((float)x[i], i);
    return;
  }
  for (uint32_t j0 = 0; j0 < s.nvec; j0 += THREADS * NV) {
    if (s.nvec > THREADS * NV) h.load(s, j0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t j = h.index(j0, i);
      if (j < s.nvec) {
        typename T::V g;
#pragma unroll
        for (int k = 0; k < T::kPer16; ++k) g[k] = (typename T::Elem)f(element<T>(h.raw[i], k), s.first(j) + k);
        if (s.whole(j)) {
          *(u32x4*)(o.base + (uint64_t)j * 16) = __builtin_bit_cast(u32x4, g);
        } else {
#pragma unroll
          for (int k = 0; k < T::kPer16; ++k)
            if (s.first(j) + k < s.v) out[s.first(j) + k] = g[k];
        }
      }
    }
  }
}

template <class T, int THREADS>
__device__ __forceinline__ void write_zeros(typename T::Elem* out, uint32_t v) {
  const Span<T> o(out, v);
  for (uint32_t j = threadIdx.x; j < o.nvec; j += THREADS) {
    if (o.whole(j)) {
      *(u32x4*)(o.base + (uint64_t)j * 16) = u32x4{0, 0, 0, 0};
    } else {
      for (uint32_t k = 0; k < T::kPer16; ++k)
        if (o.first(j) + k < v) out[o.first(j) + k] = (typename T::Elem)0.f;
    }
  }
}

// ----------------------------------------------------------- alternatives --
// Orders (logit, index): larger logits first, equal ones by index. Keys of
// different indexes differ; 0 is below every key. -0 and +0 are equal.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

struct TopShared {
  uint64_t group[kGroups];
  uint32_t rank[kGroups];
  uint64_t candidate[kCandidates];
  uint64_t wave[16];
  uint64_t bound;
  uint32_t count;
};

// How many of keys[0, n) are above `mine` (two a load: the same address for the whole wave).
__device__ __forceinline__ uint32_t above(const uint64_t* keys, uint32_t n, uint64_t mine) {
  uint32_t r = 0;
  for (uint32_t i = 0; i < n; ++i) r += keys[i] > mine;
  return r;
}

// The `top` largest of a row without NaN, largest first: emit(rank, key).
//
// The maxima of 256 groups of threads give a bound: at least `top` logits are not
// below the top-th largest of them, and about -256 ln(1 - top / 256) are. Those are
// collected, and each finds its place by counting the ones above it. Keys hold the
// index, so that ties (a constant row) do not swell the collection; where an adverse
// order does (large logits in few groups), the largest below the last one is taken
// `top` times.
template <class T, int THREADS, int NV, class F>
__device__ __forceinline__ void alternatives(const Span<T>& s, Held<T, THREADS, NV>& h, uint32_t top, TopShared& sh, F emit) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const bool again = s.nvec > THREADS * NV;
  // f(key) for the logits that this thread holds
  auto each = [&](auto f) {
    for (uint32_t j0 = 0; j0 < s.nvec; j0 += THREADS * NV) {
      if (again) h.load(s, j0);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < T::kPer16; ++k) {
          const uint32_t at = s.first(h.index(j0, i)) + k;
          f(element<T>(h.raw[i], k), at);
        }
    }
  };
  float m = -INFINITY;
  uint32_t at = ~0u;
  each([&](float x, uint32_t i) {
    if (i < s.v && (x > m || at == ~0u)) {
      m = x;
      at = i;
    }
  });
  uint64_t best = at == ~0u ? 0 : order_key(m, at);
  if (THREADS > 256) best = max64(best, __shfl_xor((unsigned long long)best, 32, 64));
  if (THREADS > 512) best = max64(best, __shfl_xor((unsigned long long)best, 16, 64));
  constexpr uint32_t kGroupsOfWave = THREADS == 256 ? 64 : THREADS == 512 ? 32 : 16;
  if (lane < kGroupsOfWave) sh.group[(tid >> 6) * kGroupsOfWave + lane] = best;
  if (tid < kGroups) sh.rank[tid] = 0;
  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  __syncthreads();
  {
    constexpr uint32_t kParts = THREADS / kGroups, kPart = kGroups / kParts;
    const uint32_t g = tid % kGroups, part = tid / kGroups;
    const uint32_t r = above(sh.group + part * kPart, kPart, sh.group[g]);
    if (kParts > 1) atomicAdd(&sh.rank[g], r);  // whole numbers: any order
    else sh.rank[g] = r;
  }
  __syncthreads();
  if (tid < kGroups && sh.rank[tid] == top - 1 && sh.group[tid]) sh.bound = sh.group[tid];
  __syncthreads();
  const uint64_t bound = sh.bound;
  const float floor = bound ? key_value(bound) : -INFINITY;
  if (m >= floor)
    each([&](float x, uint32_t i) {
      if (x >= floor && i < s.v) {
        const uint64_t key = order_key(x, i);
        if (key >= bound) {
          const uint32_t n = atomicAdd(&sh.count, 1u);
          if (n < kCandidates) sh.candidate[n] = key;
        }
      }
    });
  __syncthreads();
  const uint32_t count = sh.count;
  if (count <= kCandidates) {
    for (uint32_t n = tid; n < count; n += THREADS) {
      const uint64_t key = sh.candidate[n];
      const uint32_t r = above(sh.candidate, count, key);
      if (r < top) emit(r, key);
    }
    return;
  }
  uint64_t prev = ~0ull;
  for (uint32_t r = 0; r < top; ++r) {
    uint64_t next = 0;
    each([&](float x, uint32_t i) {
      const uint64_t key = order_key(x, i);
      if (i < s.v && key < prev && key > next) next = key;
    });
    for (int off = 32; off >= 1; off >>= 1) next = max64(next, __shfl_xor((unsigned long long)next, off, 64));
    __syncthreads();
    if (lane == 0) sh.wave[tid >> 6] = next;
    __syncthreads();
    for (uint32_t i = 0; i < THREADS / 64; ++i) next = max64(next, sh.wave[i]);
    prev = next;
    if (tid == 0) emit(r, next);
  }
}

// ---------------------------------------------------------------- kernels --
template <class T, int THREADS, int NV, bool TOP, bool GRAD>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(VocabRows a) {
  using Elem = typename T::Elem;
  __shared__ Stats<GRAD> waves[THREADS / 64];
  const uint32_t r = blockIdx.x, b = r / a.length, l = r % a.length, tid = threadIdx.x;
  const Elem* x = (const Elem*)a.logits + b * a.logits_s.batch + l * a.logits_s.row;
  Elem* g = GRAD ? (Elem*)a.grad + b * a.grad_s.batch + l * a.grad_s.row : nullptr;
  const int64_t tok = a.tokens[b * a.tokens_s.batch + l * a.tokens_s.row];
  if (tok == a.ignore) {
    if (tid == 0) {
      a.logprobs[r] = 0.f;
      a.entropy[r] = 0.f;
    }
    if (TOP && tid < (uint32_t)a.top) {
      a.top_logprobs[(int64_t)r * a.top + tid] = -INFINITY;
      a.top_tokens[(int64_t)r * a.top + tid] = -1;
    }
    if (GRAD) write_zeros<T, THREADS>(g, a.vocab);
    return;
  }
  const bool inside = tok >= 0 && tok < (int64_t)a.vocab;
  const float xt = inside ? (float)x[tok] : 0.f;
  const Span<T> s(x, a.vocab);
  Held<T, THREADS, NV> h;
  const Stats<GRAD> st = row_stats<T, THREADS, NV, true>(s, h, kLog2e, waves);
  const bool valid = st.valid();
  const float log2s = log2_hw(st.s);
  const float entropy = valid ? kLn2 * (log2s - st.t / st.s) : NAN;
  if (tid == 0) {
    a.logprobs[r] = valid && inside ? st.lnq(xt, kLog2e, 1.f) : NAN;
    a.entropy[r] = entropy;
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    float* lp = a.top_logprobs + (int64_t)r * a.top;
    int64_t* at = a.top_tokens + (int64_t)r * a.top;
    if (!valid) {
      if (tid < (uint32_t)a.top) {
        lp[tid] = NAN;
        at[tid] = -1;
      }
      return;
    }
    alternatives<T, THREADS, NV>(s, h, (uint32_t)a.top, sh, [&](uint32_t rank, uint64_t key) {
      lp[rank] = st.lnq(key_value(key), kLog2e, 1.f);
      at[rank] = (int64_t)(uint32_t)~(uint32_t)key;
    });
  }
  if constexpr (GRAD) {
    float w = a.weights ? a.weights[b * a.weights_s.batch + l * a.weights_s.row] : 0.f;
    const float u = a.entropy_weights ? a.entropy_weights[b * a.entropy_weights_s.batch + l * a.entropy_weights_s.row] : 0.f;
    if (!(valid && inside)) w = NAN;
    // d = w ([i = tok] - q) - u q (ln q + entropy), z = log2 q
    const float wu = __builtin_fmaf(u, entropy, w), ul = u * kLn2;
    write_row<T, THREADS, NV>(s, h, g, [&](float xi, uint32_t i) {
      const float z = st.y_of(xi, kLog2e) - log2s;
      const float d = -exp2_hw(z) * __builtin_fmaf(ul, fmaxf(z, -1e30f), wu);
      return i == (uint32_t)tok ? d + w : d;
    });
  }
}

struct TeacherShared {
  float w[kMaxTeacher];
  int32_t idx[kMaxTeacher];
  float total;
  int32_t bad;
};

// The teacher's softmax over its entries, by one wave: weights and tokens (-1: no
// entry) in LDS. Returns the row's loss but for the student's log sum:
// sum w (ln w - x / T) and the weights' sum.
template <class T, int THREADS, int NV, bool GRAD>
__global__ __launch_bounds__(THREADS) void topk_distill_kernel(VocabRows a) {
  using Elem = typename T::Elem;
  __shared__ Stats<GRAD> waves[THREADS / 64];
  __shared__ TeacherShared sh;
  const uint32_t r = blockIdx.x, b = r / a.length, l = r % a.length, tid = threadIdx.x, lane = tid & 63, k = (uint32_t)a.k;
  const Elem* x = (const Elem*)a.logits + b * a.logits_s.batch + l * a.logits_s.row;
  Elem* g = GRAD ? (Elem*)a.grad + b * a.grad_s.batch + l * a.grad_s.row : nullptr;
  const int64_t* tokens = a.teacher_tokens + (uint64_t)r * k;
  const float* values = a.teacher_values + (uint64_t)r * k;
  bool any = false;
  for (uint32_t j = lane; j < k; j += 64) any |= tokens[j] != -1;
  if (!__any(any)) {  // the same in every wave
    if (tid == 0) a.loss[r] = 0.f;
    if (GRAD) write_zeros<T, THREADS>(g, a.vocab);
    return;
  }
  const float inv = 1.f / a.temperature, c = kLog2e * inv;
  const float tinv = a.normalize ? inv : 1.f;
  float tm = -INFINITY, lse = 0.f;
  bool bad = false;
  if (tid < 64) {
    for (uint32_t j = lane; j < k; j += 64) {
      const int64_t i = tokens[j];
      const bool in = i >= 0 && i < (int64_t)a.vocab;
      const float t = values[j] * tinv;
      bad |= i != -1 && (!in || !(t < INFINITY));
      sh.idx[j] = in ? (int32_t)i : -1;
      sh.w[j] = in ? t : -INFINITY;
      if (in) tm = fmaxf(tm, t);
    }
    tm = reduce64(tm, Max());
    if (a.normalize) {
      float ts = 0.f;
      for (uint32_t j = lane; j < k; j += 64)
        if (sh.idx[j] >= 0) ts += exp2_hw((sh.w[j] - tm) * kLog2e);
      ts = reduce64(ts, Add());
      lse = __builtin_fmaf(kLn2, log2_hw(ts), 0.f);
      bad |= tm == -INFINITY;
    } else {
      tm = 0.f;
    }
    bad = __any(bad);
  }
  const Span<T> s(x, a.vocab);
  Held<T, THREADS, NV> h;
  const Stats<GRAD> st = row_stats<T, THREADS, NV, false>(s, h, c, waves);
  const float log2s = log2_hw(st.s);
  if (tid < 64) {
    float loss = 0.f, total = 0.f;
    for (uint32_t j = lane; j < k; j += 64) {
      const float lnw = (sh.w[j] - tm) - lse;
      const float w = sh.idx[j] >= 0 ? exp2_hw(lnw * kLog2e) : 0.f;
      if (w > 0.f) loss += w * (lnw - st.lnq((float)x[sh.idx[j]], c, inv));
      sh.w[j] = w;
      total += w;
    }
    loss = reduce64(loss, Add());
    total = reduce64(total, Add());
    bad |= !st.valid();
    if (lane == 0) {
      a.loss[r] = bad ? NAN : a.temperature * a.temperature * loss;
      sh.total = total;
      sh.bad = bad;
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    const float total = sh.total;
    const float up = sh.bad ? NAN : a.temperature * a.weights[b * a.weights_s.batch + l * a.weights_s.row];
    const float up_total = up * total;
    auto soft = [&](float xi, uint32_t) { return up_total * exp2_hw(st.y_of(xi, c) - log2s); };
    write_row<T, THREADS, NV>(s, h, g, soft);
    __syncthreads();  // the row's stores are done before its entries are written again
    for (uint32_t j = tid; j < k; j += THREADS) {
      const int32_t i = sh.idx[j];
      if (i < 0) continue;
      bool first = true;  // that names this token
      float w = 0.f;
      for (uint32_t n = 0; n < k; ++n)
        if (sh.idx[n] == i) {
          if (n < j) first = false;
          w += sh.w[n];
        }
      if (first) g[i] = (Elem)(up * (total * exp2_hw(st.y_of((float)x[i], c) - log2s) - w));
    }
  }
}

// A workgroup's size and the vectors that each thread holds, by the row's length.
template <class T, class F>
hipError_t by_length(uint32_t vocab, F launch) {
  const uint32_t nvec = (vocab + 2 * (T::kPer16 - 1)) / T::kPer16;  // the most that a row of this length spans
  if (nvec <= 256 * 4) launch(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
  else if (nvec <= 512 * 8) launch(std::integral_constant<int, 512>(), std::integral_constant<int, 8>());
  else if (nvec <= 1024 * 8) launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 8>());
  else launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
  return hipGetLastError();
}

template <class T>
hipError_t launch_logprobs(const VocabRows& a, hipStream_t st) {
  return by_length<T>(a.vocab, [&](auto threads, auto nv) {
    constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
    if (a.grad) token_logprobs_kernel<T, N, V, false, true><<<a.nrows, N, 0, st>>>(a);
    else if (a.top) token_logprobs_kernel<T, N, V, true, false><<<a.nrows, N, 0, st>>>(a);
    else token_logprobs_kernel<T, N, V, false, false><<<a.nrows, N, 0, st>>>(a);
  });
}

template <class T>
hipError_t launch_distill(const VocabRows& a, hipStream_t st) {
  return by_length<T>(a.vocab, [&](auto threads, auto nv) {
    constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
    if (a.grad) topk_distill_kernel<T, N, V, true><<<a.nrows, N, 0, st>>>(a);
    else topk_distill_kernel<T, N, V, false><<<a.nrows, N, 0, st>>>(a);
  });
}

}  // namespace

hipError_t launch_token_logprobs(int dtype, const VocabRows& a, hipStream_t st) {
  if (dtype == DZ_F32) return launch_logprobs<TypeF32>(a, st);
  return dtype == DZ_F16 ? launch_logprobs<TypeF16>(a, st) : launch_logprobs<TypeBF16>(a, st);
}

hipError_t launch_topk_distill(int dtype, const VocabRows& a, hipStream_t st) {
  if (dtype == DZ_F32) return launch_distill<TypeF32>(a, st);
  return dtype == DZ_F16 ? launch_distill<TypeF16>(a, st) : launch_distill<TypeBF16>(a, st);
}

}  // namespace dz
