// Kernels over rows of logits: log probabilities of given tokens with the
// rows' entropies and largest alternatives, the distance to a teacher's
// largest logits, and their gradients.
//
// One workgroup takes one row. What bounds these kernels is reading the row
// once (and writing its gradient once). Where only sums are asked for, the row
// streams by (stream_stats). The alternatives and the gradient need the row a second
// time: a row that fits is held in the workgroup's registers as it was read, in
// 16-byte vectors; a longer one goes by in chunks of as much, and is read again. A
// thread's vectors lie THREADS apart, so that a wave's loads cover consecutive bytes.
//
// Measured, rows of 50,272 16-bit logits: summed 4,096 of bf16 in 63 us (5.8 TB/s), with 64 alternatives
// 1,024 in 32 us (two rounds: 768 rows have a place at once, and the phases of one that is alone on its compute unit overlap
// with nothing), with a gradient 2,048 in 79-83 us (4.7-5.0 TB/s, read and written). Past the held sizes, 256 rows of
// 262,144 bf16: alternatives 57 us, gradient 77.
//
// Rows start where they start (an odd vocabulary, a view), and so do their vectors:
// loads and stores of 16 bytes at the element's alignment. The elements after the last
// whole vector are one each to the workgroup's first threads.
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
template <class T>
struct Loose16;
template <>
struct Loose16<TypeF32> {
  typedef f32x4 type __attribute__((aligned(4)));
};
template <>
struct Loose16<TypeF16> {
  typedef f16x8 type __attribute__((aligned(2)));
};
template <>
struct Loose16<TypeBF16> {
  typedef bf16x8 type __attribute__((aligned(2)));
};

template <class T>
__device__ __forceinline__ u32x4 none16() {  // no logits: -inf
  typename T::V x;
  for (int k = 0; k < T::kPer16; ++k) x[k] = (typename T::Elem)-INFINITY;
  return __builtin_bit_cast(u32x4, x);
}
template <class T>
__device__ __forceinline__ float element(const u32x4& raw, int k) {
  // bf16 by its bits: of a maximum of extended values the compiler makes an extended maximum of
  // bf16 values, which it then rounds after every step
  if (std::is_same<T, TypeBF16>::value) return __uint_as_float(k & 1 ? raw[k / 2] & 0xffff0000u : raw[k / 2] << 16);
  return (float)__builtin_bit_cast(typename T::V, raw)[k];
}
// Makes the compiler read `raw` anew, instead of keeping what an earlier pass made of it.
__device__ __forceinline__ void afresh(u32x4& raw) { asm("" : "+v"(raw)); }

// v elements at p: `full` vectors of 16 bytes, and `rem` elements.
template <class T>
struct Row {
  using Elem = typename T::Elem;
  using Loose = typename Loose16<T>::type;
  static constexpr uint32_t E = T::kPer16;
  const Elem* p;
  uint32_t v, full, rem;

  __device__ Row(const Elem* p_, uint32_t v_) : p(p_), v(v_), full(v_ / E), rem(v_ % E) {}

  // vector j0 + this thread's number: a base that is the same for the workgroup, and an offset
  __device__ __forceinline__ static auto at(const Elem* p, uint32_t j0) {
    const uint32_t offset = threadIdx.x * 16;  // of 32 bits: the base stays in scalar registers
    return (const Loose*)((const char*)(p + (uint64_t)j0 * E) + offset);
  }
  __device__ __forceinline__ u32x4 load(uint32_t j0) const { return __builtin_bit_cast(u32x4, (typename T::V)__builtin_nontemporal_load(at(p, j0))); }
  // this thread's element after the last whole vector, and its index
  __device__ __forceinline__ bool has_extra() const { return threadIdx.x < rem; }
  __device__ __forceinline__ uint32_t extra_at() const { return full * E + threadIdx.x; }
  __device__ __forceinline__ float extra() const { return has_extra() ? (float)p[extra_at()] : -INFINITY; }
};

// THREADS x NV vectors of a row from vector j0 on, in registers; -inf where there are none.
template <class T, int THREADS, int NV>
struct Held {
  static constexpr int E = T::kPer16;
  u32x4 raw[NV];

  __device__ __forceinline__ void load(const Row<T>& s, uint32_t j0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = none16<T>();
      if (j0 + i * THREADS + threadIdx.x < s.full) raw[i] = s.load(j0 + i * THREADS);
    }
  }
  __device__ __forceinline__ void load_whole(const Row<T>& s, uint32_t j0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = s.load(j0 + i * THREADS);
  }
  __device__ __forceinline__ float largest(int i) const {
    float m = element<T>(raw[i], 0);
#pragma unroll
    for (int k = 1; k < E; ++k) m = fmaxf(m, element<T>(raw[i], k));
    return m;
  }
  // The statistics with these vectors added.
  template <bool ENTROPY>
  __device__ __forceinline__ void add_to(Stats<true>& st, float c) {
    float m = st.m;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      m = fmaxf(m, largest(i));
      afresh(raw[i]);
    }
    st.rebase(m, c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      st.template add_far<ENTROPY, E>([&](int n) { return element<T>(raw[i], n); }, c);
      afresh(raw[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// A row's softmax statistics, for the whole workgroup, and the largest logit that this thread holds. Leaves
// the row in `h` where it fits.
template <class T, int THREADS, int NV, bool ENTROPY>
__device__ __forceinline__ Stats<true> row_stats(const Row<T>& s, Held<T, THREADS, NV>& h, float c, Stats<true>* waves, float& own_max) {
  auto st = Stats<true>::of(-INFINITY);
  for (uint32_t j0 = 0; j0 < s.full; j0 += THREADS * NV) {
    h.load(s, j0);
    h.template add_to<ENTROPY>(st, c);
  }
  const float extra = s.extra();
  st.rebase(fmaxf(st.m, extra), c);
  st.template add_far<ENTROPY, 1>([&](int) { return extra; }, c);
  own_max = st.m;
  return block_stats<THREADS, ENTROPY>(st, c, waves);
}

// The same where the row is not needed again: NV vectors a thread at a time, the next ones on their way while
// these are added, and the last ones from the start on. The statistics' m need not be
// the maximum: 2^y up to 2^8 do no harm, and moving it takes as long as several logits.
template <class T, int THREADS, int NV, bool ENTROPY>
__device__ __forceinline__ SoftStats stream_stats(const Row<T>& s, float c, SoftStats* waves) {
  constexpr uint32_t STEP = THREADS * NV;
  Held<T, THREADS, NV> a, b, last;
  const uint32_t whole = s.full / STEP;  // steps
  last.load(s, whole * STEP);
  auto st = SoftStats::of(-INFINITY);
  auto add = [&](Held<T, THREADS, NV>& h) {
    constexpr int N = NV * T::kPer16;
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = element<T>(h.raw[i / T::kPer16], i % T::kPer16);
      // a conversion of its own: multiply-adds that convert fp16 on the way took 72 us for 63 (4,064 rows of 50,272)
      if (std::is_same<T, TypeF16>::value) asm("" : "+v"(x[i]));
    }
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (__any(!((m - st.m) * c <= 8.f))) st.rebase(fmaxf(st.m, m), c);
    st.template add<ENTROPY, N>([&](int n) { return x[n]; }, c);
  };
  if (whole) {
    uint32_t n = 0;
    a.load_whole(s, 0);
    for (; n + 2 < whole; n += 2) {
      b.load_whole(s, (n + 1) * STEP);
      add(a);
      a.load_whole(s, (n + 2) * STEP);
      add(b);
    }
    if (n + 1 < whole) {
      b.load_whole(s, (n + 1) * STEP);
      add(a);
      add(b);
    } else {
      add(a);
    }
  }
  if (whole * STEP < s.full) add(last);
  const float extra = s.extra();
  st.rebase(fmaxf(st.m, extra), c);
  st.template add<ENTROPY, 1>([&](int) { return extra; }, c);
  return block_stats<THREADS, ENTROPY>(st, c, waves);
}

// Writes f(logit) for the whole row; `past`: without a place in the caches.
template <class T, int THREADS, int NV, class F>
__device__ __forceinline__ void write_row(const Row<T>& s, Held<T, THREADS, NV>& h, typename T::Elem* out, bool past, F f) {
  using Elem = typename T::Elem;
  using Loose = typename Row<T>::Loose;
  for (uint32_t j0 = 0; j0 < s.full; j0 += THREADS * NV) {
    if (s.full > THREADS * NV) h.load(s, j0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      typename T::V g;
#pragma unroll
      for (int k = 0; k < T::kPer16; ++k) g[k] = (Elem)f(element<T>(h.raw[i], k));
      if (j0 + i * THREADS + threadIdx.x < s.full) {
        if (past) {
          asm volatile("");  // or the compiler makes one store of the two, without the hint
          __builtin_nontemporal_store(g, (Loose*)Row<T>::at(out, j0 + i * THREADS));
          asm volatile("");
        } else {
          *(Loose*)Row<T>::at(out, j0 + i * THREADS) = g;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (s.has_extra()) out[s.extra_at()] = (Elem)f(s.extra());
}

template <class T, int THREADS>
__device__ __forceinline__ void write_zeros(typename T::Elem* out, uint32_t v) {
  const Row<T> s(out, v);
  const typename T::V zeros = __builtin_bit_cast(typename T::V, u32x4{0, 0, 0, 0});
  for (uint32_t j0 = 0; j0 + threadIdx.x < s.full; j0 += THREADS) *(typename Row<T>::Loose*)Row<T>::at(out, j0) = zeros;
  if (s.has_extra()) out[s.extra_at()] = (typename T::Elem)0.f;
}

// ----------------------------------------------------------- alternatives --
// Orders logits: the larger one has the larger key; -0 and +0 are equal. 0 is below every key.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
// Orders (logit, index): equal logits by index, the lower one first. Keys of different indexes differ.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~i; }
__device__ __forceinline__ float key_value(uint64_t k) { return value_of((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

struct TopShared {
  uint32_t group[kGroups];
  uint64_t candidate[kCandidates];
  uint64_t wave[16];
  float floor;
  uint32_t count;
};

// How many of keys[0, n) are above `mine`.
__device__ __forceinline__ uint32_t above(const uint64_t* keys, uint32_t n, uint64_t mine) {
  uint32_t r = 0;
#pragma unroll 8
  for (uint32_t i = 0; i < n; ++i) r += keys[i] > mine;
  return r;
}

// The `top` largest of a row without NaN, largest first: emit(rank, key).
//
// The maxima of 256 groups of threads give a bound: at least `top` logits are not
// below the top-th largest of them, and about -256 ln(1 - top / 256) are. Those are
// collected, and each finds its place by counting the ones above it. Where that leaves more
// than the collection holds, because many are equal to the bound (a constant row, or a mask
// that leaves fewer than `top`), those above it are collected, and then equal ones in the row's order;
// and where an adverse order puts large logits in few groups, the largest below the last one is
// taken `top` times.
template <class T, int THREADS, int NV, class F>
__device__ __forceinline__ void alternatives(const Row<T>& s, Held<T, THREADS, NV>& h, uint32_t top, float own_max, TopShared& sh, F emit) {
  constexpr int E = T::kPer16;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const bool again = s.full > THREADS * NV;
  // f(logit, index), from memory, where speed is not asked for
  auto logits = [&](auto f) {
    for (uint32_t i = tid; i < s.v; i += THREADS) f((float)s.p[i], i);
  };
  auto collect = [&](uint64_t key) {
    const uint32_t n = atomicAdd(&sh.count, 1u);
    if (n < kCandidates) sh.candidate[n] = key;
  };
  uint32_t best = order_of(own_max);
  if (THREADS > 256) best = max(best, (uint32_t)__shfl_xor((int)best, 32, 64));
  if (THREADS > 512) best = max(best, (uint32_t)__shfl_xor((int)best, 16, 64));
  constexpr uint32_t kGroupsOfWave = THREADS == 256 ? 64 : THREADS == 512 ? 32 : 16;
  if (lane < kGroupsOfWave) sh.group[(tid >> 6) * kGroupsOfWave + lane] = best;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  if (tid < 64) {
    // the top-th largest, bit by bit: the largest number that `top` groups are not below. The bits that a
    // 16-bit type does not have are 0 of positive values, and 1 in the order of negative ones.
    constexpr int kLowest = std::is_same<T, TypeBF16>::value ? 16 : std::is_same<T, TypeF16>::value ? 13 : 0;
    uint32_t k[kGroups / 64], bound = 0;
#pragma unroll
    for (uint32_t i = 0; i < kGroups / 64; ++i) k[i] = sh.group[64 * i + lane];
#pragma unroll
    for (int bit = 31; bit >= kLowest; --bit) {
      const uint32_t next = bound | (1u << bit);
      uint32_t n = 0;
#pragma unroll
      for (uint32_t i = 0; i < kGroups / 64; ++i) n += (uint32_t)__popcll(__ballot(k[i] >= next));
      if (n >= top) bound = next;
    }
    if (!(bound >> 31)) bound |= (1u << kLowest) - 1;
    if (lane == 0) sh.floor = value_of(bound);
  }
  __syncthreads();
  const float floor = sh.floor;
  for (uint32_t j0 = 0; j0 < s.full; j0 += THREADS * NV) {
    if (again) h.load(s, j0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t j = j0 + i * THREADS + tid;
      if (h.largest(i) >= floor && j < s.full) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const float x = element<T>(h.raw[i], k);
          if (x >= floor) collect(order_key(x, j * E + k));
        }
      }
    }
  }
  if (s.has_extra() && s.extra() >= floor) collect(order_key(s.extra(), s.extra_at()));
  __syncthreads();
  uint32_t count = sh.count;
  if (count > kCandidates) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    logits([&](float x, uint32_t i) {
      if (x > floor) collect(order_key(x, i));
    });
    __syncthreads();
    count = sh.count;
    for (uint32_t i0 = 0; count < top && i0 < s.v; i0 += THREADS) {  // the lowest indexes among equals
      __syncthreads();
      if (i0 + tid < s.v && (float)s.p[i0 + tid] == floor) collect(order_key(floor, i0 + tid));
      __syncthreads();
      count = sh.count;
    }
  }
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
    logits([&](float x, uint32_t i) {
      const uint64_t key = order_key(x, i);
      if (key < prev && key > next) next = key;
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
// The statistics of a row that is only read (KEEP false), or is held for a second look.
template <class T, int THREADS, int NV, bool ENTROPY, bool KEEP>
__device__ __forceinline__ Stats<KEEP> stats_of(const Row<T>& s, Held<T, THREADS, NV>& h, float c, Stats<KEEP>* waves, float& own_max) {
  if constexpr (KEEP) return row_stats<T, THREADS, NV, ENTROPY>(s, h, c, waves, own_max);
  else return stream_stats<T, THREADS, NV, ENTROPY>(s, c, waves);
}

// With alternatives, 512 threads are held to 80 registers, so that three rows share a compute unit (38 -> 35 us).
template <class T, int THREADS, int NV, bool TOP, bool GRAD>
__global__ __launch_bounds__(THREADS, TOP && THREADS == 512 ? 6 : 1) void token_logprobs_kernel(VocabRows a) {
  using Elem = typename T::Elem;
  __shared__ Stats<TOP || GRAD> waves[THREADS / 64];
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
  const Row<T> s(x, a.vocab);
  Held<T, THREADS, NV> h;
  float own_max = -INFINITY;
  const Stats<TOP || GRAD> st = stats_of<T, THREADS, NV, true, TOP || GRAD>(s, h, kLog2e, waves, own_max);
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
    alternatives<T, THREADS, NV>(s, h, (uint32_t)a.top, own_max, sh, [&](uint32_t rank, uint64_t key) {
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
    const float m0 = st.m == -INFINITY ? 0.f : st.m;
    const auto d = [&](float xi) {
      const float z = __builtin_fmaf(xi - m0, kLog2e, -log2s);
      return -exp2_hw(z) * __builtin_fmaf(ul, fmaxf(z, kLowestY), wu);
    };
    write_row<T, THREADS, NV>(s, h, g, a.past_caches, d);
    __syncthreads();  // the row's stores are done before the token's is written again
    if (tid == 0 && inside) g[tok] = (Elem)(d(xt) + w);
  }
}

struct TeacherShared {
  float w[kMaxTeacher];
  float x[kMaxTeacher];  // the student's logits of the entries
  __attribute__((aligned(16))) int32_t idx[kMaxTeacher + 4];  // -1: no entry; fours are read
  float total;
  int32_t bad;
};

// One wave makes the teacher's softmax over its entries, in LDS, before the row's statistics, and sums
// the loss after them.
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
  const float tinv = a.normalize ? inv : 1.f;  // of differences: a value at fp32's limits may leave it divided by T
  float tm = -INFINITY, lse = 0.f;
  bool bad = false;
  if (tid < 64) {
    for (uint32_t j = lane; j < k; j += 64) {
      const int64_t i = tokens[j];
      const bool in = i >= 0 && i < (int64_t)a.vocab;
      const float t = values[j];
      bad |= i != -1 && (!in || !(t < INFINITY));
      sh.idx[j] = in ? (int32_t)i : -1;
      sh.x[j] = in ? (float)x[i] : 0.f;
      sh.w[j] = in ? t : -INFINITY;
      if (in) tm = fmaxf(tm, t);
    }
    if (lane < 4) sh.idx[k + lane] = -1;
    tm = reduce64(tm, Max());
    if (a.normalize) {
      float ts = 0.f;
      for (uint32_t j = lane; j < k; j += 64)
        if (sh.idx[j] >= 0) ts += exp2_hw((sh.w[j] - tm) * tinv * kLog2e);
      ts = reduce64(ts, Add());
      lse = kLn2 * log2_hw(ts);
      bad |= tm == -INFINITY;
    } else {
      tm = 0.f;
    }
    bad = __any(bad);
  }
  const Row<T> s(x, a.vocab);
  Held<T, THREADS, NV> h;
  float own_max = -INFINITY;
  const Stats<GRAD> st = stats_of<T, THREADS, NV, false, GRAD>(s, h, c, waves, own_max);
  const float log2s = log2_hw(st.s);
  if (tid < 64) {
    float loss = 0.f, far = 0.f, total = 0.f;
    for (uint32_t j = lane; j < k; j += 64) {
      const float lnw = (sh.w[j] - tm) * tinv - lse;
      const float w = sh.idx[j] >= 0 ? exp2_hw(lnw * kLog2e) : 0.f;
      if (w > 0.f) {
        const float lnq = st.lnq(sh.x[j], c, inv);
        // a logit of the type's lowest value, which a temperature below 1, or a largest one at the other end, takes
        // past fp32's range: beside it nothing else counts, and its distance is taken undivided, weight by weight
        if (lnq == -INFINITY) far += w * st.m - w * sh.x[j];
        else loss += w * (lnw - lnq);
      }
      sh.w[j] = w;
      total += w;
    }
    loss = reduce64(loss, Add());
    far = reduce64(far, Add());
    total = reduce64(total, Add());
    bad |= !st.valid();
    if (lane == 0) {
      a.loss[r] = bad ? NAN : a.temperature * a.temperature * loss + a.temperature * far;
      sh.total = total;
      sh.bad = bad;
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    const float total = sh.total;
    const float up = sh.bad ? NAN : a.temperature * a.weights[b * a.weights_s.batch + l * a.weights_s.row];
    const float up_total = up * total;
    const float m0 = st.m == -INFINITY ? 0.f : st.m;
    const auto soft = [&](float xi) { return up_total * exp2_hw(__builtin_fmaf(xi - m0, c, -log2s)); };
    write_row<T, THREADS, NV>(s, h, g, a.past_caches, soft);
    __syncthreads();  // the row's stores are done before its entries are written again
    for (uint32_t j = tid; j < k; j += THREADS) {
      const int32_t i = sh.idx[j];
      if (i < 0) continue;
      bool first = true;  // that names this token
      float w = sh.w[j];
#pragma unroll 4
      for (uint32_t n = 0; n < k; n += 4) {
        const i32x4 four = *(const i32x4*)(sh.idx + n);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          if (four[e] == i && n + e != j) {
            if (n + e < j) first = false;
            w += sh.w[n + e];
          }
      }
      if (first) g[i] = (Elem)(up * (total * exp2_hw(__builtin_fmaf(sh.x[j] - m0, c, -log2s)) - w));
    }
  }
}

// A workgroup's size and the vectors that each thread holds, by the row's length: steps of a factor of 2 to 1.25, and
// workgroups of which two or three share a compute unit, so that one's loads overlap another's sums. (Short rows leave
// most of the smallest size empty: 4,096 rows of 1,000 fp16 with gradient take 25 us, of which the bytes are 3.)
template <class T, class F>
hipError_t by_length(uint32_t vocab, F launch) {
  const uint32_t nvec = vocab / T::kPer16;
  if (nvec <= 256 * 8) launch(std::integral_constant<int, 256>(), std::integral_constant<int, 8>());
  else if (nvec <= 512 * 8) launch(std::integral_constant<int, 512>(), std::integral_constant<int, 8>());
  else if (nvec <= 512 * 13) launch(std::integral_constant<int, 512>(), std::integral_constant<int, 13>());
  else if (nvec <= 1024 * 8) launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 8>());
  else if (nvec <= 1024 * 13) launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 13>());
  else launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
  return hipGetLastError();
}

// The same where the row streams by: 256 threads, of which 8 workgroups share a compute unit; 1,024
// where there are fewer rows than compute units, and each has one to itself.
template <class F>
hipError_t by_rows(uint32_t nrows, uint32_t vocab, F launch) {
  if (nrows <= 256 && vocab > 8192) launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
  else launch(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
  return hipGetLastError();
}

// Gradients that the 256 MB Infinity Cache does not hold together with their logits are stored past the
// caches: 2,048 rows of 50,272 bf16 93 -> 83 us, where every call has another gradient; 128 MB of fp32 that
// are written over again and again 45 us without, 51 with.
template <class T>
bool past_caches(const VocabRows& a) {
  return 2 * (uint64_t)a.nrows * a.vocab * sizeof(typename T::Elem) > (256u << 20);
}

template <class T>
hipError_t launch_logprobs(VocabRows a, hipStream_t st) {
  a.past_caches = past_caches<T>(a);
  if (!a.grad && !a.top)
    return by_rows(a.nrows, a.vocab, [&](auto threads, auto nv) {
      constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
      token_logprobs_kernel<T, N, V, false, false><<<a.nrows, N, 0, st>>>(a);
    });
  return by_length<T>(a.vocab, [&](auto threads, auto nv) {
    constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
    if (a.grad) token_logprobs_kernel<T, N, V, false, true><<<a.nrows, N, 0, st>>>(a);
    else token_logprobs_kernel<T, N, V, true, false><<<a.nrows, N, 0, st>>>(a);
  });
}

template <class T>
hipError_t launch_distill(VocabRows a, hipStream_t st) {
  a.past_caches = past_caches<T>(a);
  if (!a.grad)
    return by_rows(a.nrows, a.vocab, [&](auto threads, auto nv) {
      constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
      topk_distill_kernel<T, N, V, false><<<a.nrows, N, 0, st>>>(a);
    });
  return by_length<T>(a.vocab, [&](auto threads, auto nv) {
    constexpr int N = decltype(threads)::value, V = decltype(nv)::value;
    topk_distill_kernel<T, N, V, true><<<a.nrows, N, 0, st>>>(a);
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
