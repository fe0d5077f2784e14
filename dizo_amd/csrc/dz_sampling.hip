// One token of each row of logits, from a given uniform number.
//
// Weights w = exp((x - max) / T). top-k keeps the k largest, top-p the fewest of these, largest first, whose
// weights reach p of their sum, min-p those of at least min_p (the largest weight is 1); equal logits in the order of
// their tokens. All three keep a beginning of the row sorted by size, so what is kept is a logit, the cut, with
// everything above it and the first few that equal it. The token is the first, by number, up to which the kept weights
// exceed u of their sum.
//
// Sums decide which token comes out, so they must not depend on who adds first, and an error of 2^-24 (fp32's) next to one
// of 50,000 borders would give another token in one of a few thousand rows. Weights are computed in 64 bits and
// kept as whole numbers of 2^-46 (2^-42 for the largest vocabularies, so that a row's sum fits 64 bits): sums are exact in any
// order, and a token of less weight than half of that, which one number of 2^24 could hardly reach, is not drawn.
//
// A workgroup takes a row. The row is read once and held in LDS (512 x 32,003 fp32: 65 us, read again for each pass 71), then gone through:
// sums of weights by bins of their distance to the largest (top-p), the logits of the bin that the cut lies in, sorted; and sums of what is
// kept by pieces of the row. Top-k sorts the few logits that can matter and needs none of that. What bounds it: the vector
// units (weights in 64 bits: about 20 operations each, twice a logit), then the chain of phases: 17 us for one row of 50,272
// with top-k, 65 for 512 x 32,003 with top-p, two rounds of rows; a read of the logits alone would take 13.
#include "dz_sampling.h"
#include "dz_token_math.h"

namespace dz {
namespace {

constexpr int kBins = 2048;
constexpr int kPowers = 1024;
constexpr int kBinBits = 5;  // a bin is 2^kBinBits places: 32 bins for each power of two, 48 of which a weight can have
constexpr int kHeldBytes = 128 * 1024;  // of a row in LDS

// The order of logits: a logit's key, and its token from the last on. Larger first, equal ones by token.
__device__ __forceinline__ uint32_t token_of(uint64_t low) { return ~(uint32_t)low; }
__device__ __forceinline__ uint64_t order_of(uint32_t key, uint32_t token) { return (uint64_t)key << 32 | (uint32_t)~token; }

template <int THREADS, int PIECES>
struct Shared {
  static constexpr int kThreads = THREADS, kWaves = THREADS / 64;
  static constexpr int kList = THREADS;  // logits that are sorted one by one
  union {  // sums by bins, then what one of them holds
    uint64_t bins[kBins];
    uint64_t list[kList];
  };
  uint64_t pieces[PIECES];  // sums of a wave's part of a slab
  double powers[kPowers];  // 2^(i / kPowers - 2)
  uint64_t wave_sum[kWaves];
  float wave_max[kWaves];
  uint32_t wave_flag[kWaves];
  uint64_t found_before;
  uint64_t cut;
  uint32_t found, low, high, listed;
  uint32_t edge[2];  // logits between which something lies, as keys
};

// fp32 numbers as whole ones of the same order. (-0 equals 0.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Sums up to and with this lane: of 24, 24 and 16 bits each, whose sums over 64 lanes fit 32. SHORT: of numbers up to 2^49 (8 weights),
// of 24 and 25 bits.
__device__ __forceinline__ uint32_t wave_scan_part(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // the lane before, of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 to the second 16 lanes, and the third's last to the fourth
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}
template <bool SHORT>
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {
  const uint32_t low = wave_scan_part((uint32_t)x & 0xffffff);
  if (SHORT) return low + ((uint64_t)wave_scan_part((uint32_t)(x >> 24)) << 24);
  const uint32_t middle = wave_scan_part((uint32_t)(x >> 24) & 0xffffff), high = wave_scan_part((uint32_t)(x >> 48));
  return low + ((uint64_t)middle << 24) + ((uint64_t)high << 48);
}

// Sums up to and with this thread, and of all of them. Every thread has read what the last call left.
template <class Sh>
__device__ __forceinline__ uint64_t block_scan(Sh& sh, uint64_t x, uint64_t& all) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_scan<false>(x);
  __syncthreads();
  if (lane == 63) sh.wave_sum[wave] = x;
  __syncthreads();
  all = 0;
  for (uint32_t i = 0; i < Sh::kWaves; ++i) {
    if (i < wave) x += sh.wave_sum[i];
    all += sh.wave_sum[i];
  }
  return x;
}

// The first of n places whose sum with all before it reaches `target` (at least 1), and the sum before it: found and
// found_before. n where none does.
template <class Sh>
__device__ __forceinline__ void find(Sh& sh, const uint64_t* values, uint32_t n, uint64_t target) {
  const uint32_t tid = threadIdx.x, each = (n + Sh::kThreads - 1) / Sh::kThreads;
  uint64_t mine = 0, all;
  for (uint32_t i = 0; i < each; ++i)
    if (tid * each + i < n) mine += values[tid * each + i];
  uint64_t before = block_scan(sh, mine, all) - mine;
  if (tid == 0 && all < target) {
    sh.found = n;
    sh.found_before = all;
  }
  if (before < target && before + mine >= target) {
    for (uint32_t i = 0; i < each; ++i) {
      const uint64_t v = tid * each + i < n ? values[tid * each + i] : 0;
      if (before + v >= target) {
        sh.found = tid * each + i;
        sh.found_before = before;
        break;
      }
      before += v;
    }
  }
  __syncthreads();
}

// A row, 16 bytes a thread and slab: HELD in LDS, or read again for each pass.
template <class T, bool HELD, int kThreads>
struct Row {
  typedef typename T::V Loose __attribute__((aligned(sizeof(typename T::Elem))));
  using Elem = typename T::Elem;
  static constexpr int PER = T::kPer16;
  const Elem* x;
  typename T::V* held;  // slab after slab
  uint32_t vocab, slabs;
  bool infinite;  // the largest logit is +inf: those are 0, the others -inf

  __device__ __forceinline__ typename T::V load(uint32_t s) const {  // those past the row are -inf
    const uint32_t at = (s * kThreads + threadIdx.x) * PER;
    typename T::V v;
    if (at + PER <= vocab) {
      v = *(const Loose*)(x + at);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = at + j < vocab ? x[at + j] : (Elem)-INFINITY;
    }
    return v;
  }
  // f(the logits of the thread's vector of a slab, the first one's token)
  template <class F>
  __device__ __forceinline__ void give(const typename T::V& e, uint32_t s, F f) const {
    float v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = (float)e[j];
    if (infinite)
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
    f(v, (s * kThreads + threadIdx.x) * PER);
  }
  template <class F>
  __device__ __forceinline__ void slab(uint32_t s, F f) const {
    give(HELD ? held[s * kThreads + threadIdx.x] : load(s), s, f);
  }
  // for each slab: f(s, logits, first token)
  template <class F>
  __device__ __forceinline__ void slabs_do(F f) const {
#pragma unroll 1
    for (uint32_t s = 0; s < slabs; ++s) slab(s, [&](const float(&v)[PER], uint32_t at) { f(s, v, at); });
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    slabs_do([&](uint32_t, const float(&v)[PER], uint32_t at) {
#pragma unroll
      for (int j = 0; j < PER; ++j) f(v[j], at + j);
    });
  }
  // The first pass: four slabs' loads at a time.
  template <class F>
  __device__ __forceinline__ void first(F f) const {
    for (uint32_t s0 = 0; s0 < slabs; s0 += 4) {
      typename T::V e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i < slabs) e[i] = load(s0 + i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i < slabs) {
          if (HELD) held[(s0 + i) * kThreads + threadIdx.x] = e[i];
#pragma unroll
          for (int j = 0; j < PER; j += 2) f((float)e[i][j], (float)e[i][j + 1]);
        }
    }
  }
};

// Sorts 2^i >= n numbers, one a thread, the largest first.
template <class Sh>
__device__ __forceinline__ void sort(Sh& sh, uint64_t& e, uint32_t n) {
  const uint32_t tid = threadIdx.x;
  uint32_t size = 2;
  while (size < n) size *= 2;
  if (n <= 64 && tid >= 64) return;  // (no barrier then)
  for (uint32_t k = 2; k <= size; k *= 2)
    for (uint32_t j = k / 2; j > 0; j /= 2) {
      uint64_t o;
      if (j >= 64) {
        __syncthreads();
        sh.list[tid] = e;
        __syncthreads();
        o = sh.list[tid ^ j];
      } else {
        o = __shfl_xor(e, j);
      }
      const bool first = (tid & j) == 0, down = (tid & k) == 0;  // the larger one goes first
      if (first == down ? o > e : o < e) e = o;
    }
}

// What is kept: logits whose order is the cut's or above it.
template <class T, bool HELD, int kThreads>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleRows a) {
  constexpr int PER = T::kPer16, kWaves = kThreads / 64, kList = kThreads;
  __shared__ Shared<kThreads, HELD ? kHeldBytes / 1024 : kMaxSampleVocab / PER / 64> sh;
  extern __shared__ __attribute__((aligned(16))) char held[];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
  Row<T, HELD, kThreads> row;
  row.x = (const typename T::Elem*)a.logits + (int64_t)r * a.stride;
  row.vocab = a.vocab;
  row.slabs = (a.vocab + kThreads * PER - 1) / (kThreads * PER);
  row.infinite = false;
  row.held = (typename T::V*)held;
  const float u = a.uniform[r];
  const double temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  const double top_p = a.top_ps ? a.top_ps[r] : a.top_p, min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  const int32_t row_k = a.top_ks ? a.top_ks[r] : a.top_k, top_k = temperature == 0 ? 1 : row_k;
  const double unit = temperature == 0 ? 1.0 : temperature;

  for (int i = tid; i < kPowers; i += kThreads) sh.powers[i] = exp2(i / (double)kPowers - 2.0);
  for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
  if (tid == 0) sh.listed = 0;
  bool none = !(u >= 0.f && u <= 1.f) || !(temperature == 0 || (temperature >= 0x1p-63 && temperature < 0x1p64)) || row_k < 0 ||
              !(top_p >= 0 && top_p <= 1) || !(min_p >= 0 && min_p <= 1);
  float mine = -INFINITY;  // the largest of this thread's
  row.first([&](float x, float y) {
    mine = fmaxf(fmaxf(mine, x), y);
    none |= __builtin_isunordered(x, y);
  });
  float m = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  none = __any(none);
  if (lane == 0) {
    sh.wave_max[wave] = m;
    sh.wave_flag[wave] = none;
  }
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) {
    m = fmaxf(m, sh.wave_max[i]);
    none |= sh.wave_flag[i] != 0;
  }
  if (none || m == -INFINITY) {  // no distribution
    if (tid == 0) a.tokens[r] = -1;
    return;
  }
  if (m == INFINITY) {
    row.infinite = true;
    mine = mine == INFINITY ? 0.f : -INFINITY;
    m = 0.f;
  }

  // Weights as whole numbers of 2^-shift. A logit's place is its distance to 2^-2 of that, in 1,024ths of a power of two (and 0 below):
  // place n + f gives 2^(n / 1024 - 2) 2^(f / 1024), by a table, and by Taylor's polynomial (the next term is under 2^-46.6 of
  // it). Places are exact to 2^-38, which moves a weight by 2^-48 of it.
  const int lg = 32 - __clz((a.vocab - 1) | 1), shift = 62 - lg < 46 ? 62 - lg : 46;
  constexpr double kLn = 0x1.62e42fefa39efp-11;  // ln 2 / 1024
  const double per = kPowers * 1.4426950408889634074 / unit, wide_m = m, most = kPowers * (double)(shift + 2);
  auto place_of = [&](float x) { return fmax(__builtin_fma((double)x - wide_m, per, most), 0.0); };
  auto weight_at = [&](double place) -> uint64_t {
    const uint32_t n = (uint32_t)place;
    const double f = __builtin_amdgcn_fract(place);
    double p = __builtin_fma(f, kLn * kLn * kLn / 6, kLn * kLn / 2);
    p = __builtin_fma(f, p, kLn) * f;
    const double w = sh.powers[n % kPowers], y = __builtin_fma(w, p, w);
    const double scaled = __hiloint2double(__double2hiint(y) + (int32_t)(n / kPowers << 20), __double2loint(y));
    return (uint64_t)__double_as_longlong(scaled + 0x1p52) & 0xfffffffffffffull;
  };
  auto weight = [&](float x) -> uint64_t { return weight_at(place_of(x)); };
  // The least number (as a key) whose place reaches `place`; the largest logit's does. A wave at a time: by the place's inverse, to within a
// few numbers where their steps are not too small for it, and otherwise in 64ths of what is left.
  auto least_reaching = [&](double place) -> uint32_t {
    auto reaches = [&](uint32_t k) { return place_of(of_key(k)) >= place; };
    uint32_t low = key_of(-INFINITY), high = key_of(m);
    if (!(place > 0.0)) return low;
    const uint32_t near = key_of((float)__builtin_fma((place - most) * kLn, unit, wide_m));
    uint32_t k = near - 32 + lane;
    uint64_t reached = __ballot(k < low ? false : k > high ? true : reaches(k));
    if (reached >> 63 && !(reached & 1)) return near - 32 + __builtin_ctzll(reached);
    while (low < high) {
      const uint32_t step = (high - low) / 64 + 1;
      k = lane < (high - low) / step ? low + lane * step : high;
      reached = __ballot(reaches(k));
      const uint32_t first = __builtin_ctzll(reached);  // (high reaches it)
      high = __builtin_amdgcn_readlane(k, first);
      if (first) low = __builtin_amdgcn_readlane(k, first - 1) + 1;
      if (!first) break;
    }
    return high;
  };
  // min_p as the least logit that it keeps; the largest is always kept
  const double least_place = min_p > 0 ? kPowers * (log2(min_p) + (shift + 2)) : 0.0;

  auto clear = [&]() {
    for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
  };
  auto add_to = [&](uint32_t bin, uint64_t value) { atomicAdd((unsigned long long*)&sh.bins[bin], (unsigned long long)value); };
  // Bins by the distance to the largest in places.
  const uint32_t top_place = (uint32_t)most;
  auto bin_of = [&](float x) { return (top_place - (uint32_t)place_of(x)) >> kBinBits; };
  // The least logit of a bin, as a key.
  auto least_of = [&](uint32_t bin) { return least_reaching((double)top_place - (double)((bin << kBinBits) + (1 << kBinBits) - 1)); };
  // Logits (above -inf) from `from` to below `below` of an order of `least` or above, one a thread and sorted; the others are 0 (of no
  // order). How many: more than kList if they do not fit, and nothing then.
  uint64_t e;
  auto weight_of = [&](uint64_t order) -> uint64_t { return order ? weight(of_key((uint32_t)(order >> 32))) : 0; };
  auto list = [&](float from, float below, uint64_t least) -> uint32_t {
    __syncthreads();
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    row.slabs_do([&](uint32_t, const float(&v)[PER], uint32_t token) {
      bool some = false;
#pragma unroll
      for (int j = 0; j < PER; ++j) some |= v[j] >= from && v[j] < below;
      if (!some) return;  // (nearly all)
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (!(v[j] >= from && v[j] < below) || v[j] == -INFINITY) continue;
        const uint64_t order = order_of(key_of(v[j]), token + j);
        if (order < least) continue;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kList) sh.list[at] = order;
      }
    });
    __syncthreads();
    const uint32_t n = sh.listed;
    e = 0;
    if (n <= kList) {
      if (tid < n) e = sh.list[tid];
      sort(sh, e, n);
    }
    return n;
  };
  // The order at which the values of the logits of an order of `least` or above, summed from the largest on, reach `target`; sh.bins
  // has the sums by distance. 0: they do not.
  auto cut_at = [&](uint64_t target, uint64_t least, bool counts) -> uint64_t {
    auto value = [&](float x) -> uint64_t { return counts ? 1 : weight(x); };
    find(sh, sh.bins, kBins, target);
    const uint32_t bin = sh.found;
    uint64_t before = sh.found_before;
    if (bin == kBins) return least;
    if (wave < 2) {
      const uint32_t k = wave == 0 ? least_of(bin) : bin ? least_of(bin - 1) : key_of(INFINITY);
      if (lane == 0) sh.edge[wave] = k;
    }
    __syncthreads();
    const float from = of_key(sh.edge[0]), below = of_key(sh.edge[1]);
    auto in_bin = [&](float x) { return x >= from && x < below; };
    if (list(from, below, least) <= kList) {
      uint64_t all;
      const uint64_t v = counts ? e != 0 : weight_of(e), upto = block_scan(sh, v, all);
      if (before + upto - v < target && before + upto >= target) sh.cut = e;
      __syncthreads();
      return sh.cut;
    }
    // Too many for that: bins of keys, down to one key, and the first of those that have it by their token.
    uint32_t low = ~0u, high = 0;
    if (tid == 0) {
      sh.low = ~0u;
      sh.high = 0;
    }
    __syncthreads();
    auto of_bin = [&](float x, uint32_t token) { return in_bin(x) && x != -INFINITY && order_of(key_of(x), token) >= least; };
    row.each([&](float x, uint32_t token) {
      if (of_bin(x, token)) {
        const uint32_t k = key_of(x);
        low = k < low ? k : low;
        high = k > high ? k : high;
      }
    });
    if (low <= high) {
      atomicMin(&sh.low, low);
      atomicMax(&sh.high, high);
    }
    __syncthreads();
    low = sh.low;
    high = sh.high;
    while (low < high) {
      const int bits = 32 - __clz(high - low), s = bits > 11 ? bits - 11 : 0;
      __syncthreads();
      clear();
      __syncthreads();
      row.each([&](float x, uint32_t token) {
        const uint32_t k = key_of(x);
        if (k >= low && k <= high && of_bin(x, token)) add_to((high - k) >> s, value(x));
      });
      __syncthreads();
      find(sh, sh.bins, kBins, target - before);
      if (sh.found >= kBins) break;  // (the sums are the ones that found the bin)
      before += sh.found_before;
      high = high - (sh.found << s);
      low = high - low < (1u << s) - 1 ? low : high - ((1u << s) - 1);
    }
    const uint64_t one = value(of_key(low)), nth = (target - before + one - 1) / one;  // of those equal to the cut
    auto is_equal = [&](float x, uint32_t token) { return x != -INFINITY && key_of(x) == low && order_of(low, token) >= least; };
    __syncthreads();
    row.slabs_do([&](uint32_t s, const float(&v)[PER], uint32_t at) {
      uint64_t n = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) n += is_equal(v[j], at + j);
      n = wave_scan<true>(n);
      if (lane == 63) sh.pieces[s * kWaves + wave] = n;
    });
    __syncthreads();
    find(sh, sh.pieces, row.slabs * kWaves, nth);
    const uint32_t piece = sh.found;
    if (piece < row.slabs * kWaves && wave == piece % kWaves) {
      row.slab(piece / kWaves, [&](const float(&v)[PER], uint32_t at) {
        uint64_t n = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) n += is_equal(v[j], at + j);
        uint64_t upto = sh.found_before + wave_scan<true>(n) - n;
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (is_equal(v[j], at + j) && ++upto == nth) sh.cut = order_of(low, at + j);
      });
    }
    __syncthreads();
    return sh.cut;
  };
  // What is not below an order, nor below a logit: of tokens before `end` what reaches `from`, of later ones what reaches `after`.
  struct Kept {
    float cut, from, after;
    uint32_t end;
  };
  auto kept_of = [](uint64_t order, float least) {
    if (!order) return Kept{-INFINITY, least, least, 0};
    const uint32_t key = (uint32_t)(order >> 32);
    return Kept{of_key(key), fmaxf(of_key(key), least), fmaxf(of_key(key + 1), least), token_of(order) + 1};
  };
  // For a vector of logits, which of them the two are.
  auto bound = [&](const Kept& k, float(&v)[PER], uint32_t at) {
    if (at < k.end && at + PER > k.end) {  // (one vector of the row)
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (at + j >= k.end && v[j] == k.cut) v[j] = -INFINITY;
    }
    return at < k.end ? k.from : k.after;
  };
  // What top-p keeps of a sum: whole numbers that have to be reached.
  auto share_of = [&](uint64_t total) -> uint64_t {
    const double share = __builtin_ceil(top_p * (double)total);
    return share < 1.0 ? 1 : (uint64_t)share;
  };
  // u of a sum, as what has to be reached.
  auto drawn_of = [&](uint64_t sum) -> uint64_t {
    const uint64_t target = (uint64_t)__builtin_floor((double)u * (double)sum) + 1;
    return target < sum ? target : sum;
  };

  uint64_t cut = 0;
  if (top_k > 0 && (uint32_t)top_k < a.vocab) {
    // The bin up to which top_k threads have their largest holds top_k logits, too: nothing further away is among the largest.
    uint32_t last_bin = kBins;
    if (top_k <= kThreads) {
      if (mine != -INFINITY) add_to(bin_of(mine), 1);
      __syncthreads();
      find(sh, sh.bins, kBins, top_k);
      last_bin = sh.found;
      const uint32_t k = last_bin < kBins && wave == 0 ? least_of(last_bin) : key_of(-INFINITY);
      if (tid == 0) sh.edge[0] = k;
      __syncthreads();
    }
    const uint32_t n = top_k <= kThreads ? list(of_key(sh.edge[0]), INFINITY, 0) : kList + 1;
    if (n <= kList) {
      // All that matters is in the list, sorted: what is kept is its beginning.
      uint64_t total, sum;
      if (tid >= (uint32_t)top_k) e = 0;
      if (top_p < 1.0) {
        const uint64_t w = weight_of(e), before = block_scan(sh, w, total) - w;
        if (before >= share_of(total)) e = 0;
      }
      if (e && place_of(of_key((uint32_t)(e >> 32))) < least_place) e = 0;
      const uint32_t kept = __syncthreads_count(e != 0);
      e = e << 32 | e >> 32;  // by token from here on
      sort(sh, e, kept);
      const uint64_t w = weight_of(e << 32 | e >> 32), before = block_scan(sh, w, sum) - w, target = drawn_of(sum);
      if (before < target && before + w >= target) a.tokens[r] = token_of(e >> 32);
      return;
    }
    __syncthreads();
    clear();
    __syncthreads();
    row.each([&](float x, uint32_t) {
      if (x != -INFINITY && bin_of(x) <= last_bin) add_to(bin_of(x), 1);
    });
    __syncthreads();
    cut = cut_at(top_k, 0, true);
    __syncthreads();
    clear();
    __syncthreads();
  }
  if (top_p < 1.0) {
    const Kept kept = kept_of(cut, -INFINITY);
    row.slabs_do([&](uint32_t, const float(&v)[PER], uint32_t at) {
      float x[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = v[j];
      const float from = bound(kept, x, at);
      uint64_t w[PER];
      uint32_t bin[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double place = place_of(x[j]);
        w[j] = weight_at(place);
        bin[j] = (top_place - (uint32_t)place) >> kBinBits;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (w[j] && x[j] >= from) add_to(bin[j], w[j]);
    });
    __syncthreads();
    uint64_t sum = 0, total;
    for (int i = tid; i < kBins; i += kThreads) sum += sh.bins[i];
    block_scan(sh, sum, total);
    cut = cut_at(share_of(total), cut, false);
  }

  // What is kept of each piece of the row, and the piece and token that u falls on.
  if (wave == 0) {
    const uint32_t k = least_reaching(least_place);
    if (lane == 0) sh.edge[0] = k;
  }
  __syncthreads();
  const Kept kept = kept_of(cut, of_key(sh.edge[0]));
  auto kept_weights = [&](const float(&v)[PER], uint32_t at, uint64_t(&w)[PER]) {
    float x[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = v[j];
    const float from = bound(kept, x, at);
    bool some = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      some |= x[j] >= from;
      w[j] = 0;
    }
    if (!some) return;  // (where little is kept, all of most waves')
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint64_t one = weight(x[j]);
      w[j] = x[j] >= from ? one : 0;
    }
  };
  const uint32_t pieces = row.slabs * kWaves;
  uint64_t all = 0, sum;
  row.slabs_do([&](uint32_t s, const float(&v)[PER], uint32_t at) {
    uint64_t w[PER], n = 0;
    kept_weights(v, at, w);
#pragma unroll
    for (int j = 0; j < PER; ++j) n += w[j];
    all += n;
    n = wave_scan<true>(n);
    if (lane == 63 && s < row.slabs) sh.pieces[s * kWaves + wave] = n;
  });
  block_scan(sh, all, sum);
  const uint64_t target = drawn_of(sum);
  find(sh, sh.pieces, pieces, target);
  const uint32_t piece = sh.found;
  if (piece < pieces && wave == piece % kWaves) {
    row.slab(piece / kWaves, [&](const float(&v)[PER], uint32_t at) {
      uint64_t w[PER], n = 0;
      kept_weights(v, at, w);
#pragma unroll
      for (int j = 0; j < PER; ++j) n += w[j];
      uint64_t before = sh.found_before + wave_scan<true>(n) - n;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (before < target && before + w[j] >= target) a.tokens[r] = at + j;
        before += w[j];
      }
    });
  }
}

template <class T, int THREADS>
hipError_t launch_held(const SampleRows& a, hipStream_t st) {
  const uint32_t slab = THREADS * 16, bytes = (a.vocab * (16 / T::kPer16) + slab - 1) / slab * slab;
  const hipError_t e = hipFuncSetAttribute((const void*)sample_kernel<T, true, THREADS>, hipFuncAttributeMaxDynamicSharedMemorySize, kHeldBytes);
  if (e != hipSuccess) return e;
  sample_kernel<T, true, THREADS><<<a.nrows, THREADS, bytes, st>>>(a);
  return hipGetLastError();
}
// Threads by the row: 1,024 where its LDS leaves room for one workgroup a compute unit; 512 where two find room (512 x 16,384 bf16, top-p:
// 28 us, 1,024 threads 40; at 32,000 65 and 64); 256 for rows of up to 4,096 where there are many (2,000 x 4,096: 35 us, 512 threads 42;
// 256 x 4,096: 13.8 and 12.7) and of up to 2,048.
template <class T>
hipError_t launch_typed(const SampleRows& a, hipStream_t st) {
  const uint32_t bytes = a.vocab * (16 / T::kPer16);
  if (a.vocab <= (a.nrows > 512 ? 4096u : 2048u)) return launch_held<T, 256>(a, st);
  if (bytes <= 48 * 1024) return launch_held<T, 512>(a, st);
  if (bytes <= kHeldBytes) return launch_held<T, 1024>(a, st);
  sample_kernel<T, false, 1024><<<a.nrows, 1024, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(int dtype, const SampleRows& a, hipStream_t st) {
  switch (dtype) {
    case 0: return launch_typed<TypeF32>(a, st);
    case 1: return launch_typed<TypeF16>(a, st);
    default: return launch_typed<TypeBF16>(a, st);
  }
}

}  // namespace dz
