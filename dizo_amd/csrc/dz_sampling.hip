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
#include "dz_sampling.h"
#include "dz_token_math.h"

namespace dz {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;
constexpr int kMaxPieces = (int)(kMaxSampleVocab / (kThreads * 4)) * kWaves;  // a wave's part of 1,024 vectors

struct Shared {
  uint64_t bins[kBins];
  uint64_t pieces[kMaxPieces];
  uint64_t wave_sum[kWaves];
  float wave_max[kWaves];
  uint32_t wave_flag[kWaves];
  uint64_t found_before;
  uint32_t found, low, high, token;
};

// fp32 numbers as whole ones of the same order. (-0 equals 0.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {  // sums up to and with this lane
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_up(x, d);
    if (lane >= (uint32_t)d) x += o;
  }
  return x;
}

// The first of n places whose sum with all before it reaches `target` (at least 1), and the sum before it: found and
// found_before. n where none does.
__device__ __forceinline__ void find(Shared& sh, const uint64_t* values, uint32_t n, uint64_t target) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, each = (n + kThreads - 1) / kThreads;
  uint64_t mine = 0;
  for (uint32_t i = 0; i < each; ++i)
    if (tid * each + i < n) mine += values[tid * each + i];
  const uint64_t upto = wave_scan(mine);
  if (lane == 63) sh.wave_sum[wave] = upto;
  if (tid == 0) {
    sh.found = n;
    sh.found_before = 0;
  }
  __syncthreads();
  uint64_t before = upto - mine;
  for (uint32_t i = 0; i < wave; ++i) before += sh.wave_sum[i];
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

template <class T>
struct Row {
  typedef typename T::V Loose __attribute__((aligned(sizeof(typename T::Elem))));
  static constexpr int PER = T::kPer16;
  const typename T::Elem* x;
  uint32_t vocab, slabs;
  bool infinite;  // the largest logit is +inf: those are 0, the others -inf

  // f(logits of the thread's vector of a slab, the first one's token); those past the row are -inf
  template <class F>
  __device__ __forceinline__ void slab(uint32_t s, F f) const {
    const uint32_t at = (s * kThreads + threadIdx.x) * PER;
    float v[PER];
    if (at + PER <= vocab) {
      const typename T::V e = *(const Loose*)(x + at);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = (float)e[j];
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = at + j < vocab ? (float)x[at + j] : -INFINITY;
    }
    if (infinite)
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
    f(v, at);
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (uint32_t s = 0; s < slabs; ++s) slab(s, [&](const float(&v)[PER], uint32_t) {
#pragma unroll
      for (int j = 0; j < PER; ++j) f(v[j]);
    });
  }
};

// What is kept: logits above the cut's, and the first `equal` of those that equal it.
struct Cut {
  uint32_t key, equal;
  uint32_t there;  // that equal it
};

template <class T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleRows a) {
  __shared__ Shared sh;
  constexpr int PER = Row<T>::PER;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
  Row<T> row{(const typename T::Elem*)a.logits + (int64_t)r * a.stride, a.vocab, (a.vocab + kThreads * PER - 1) / (kThreads * PER), false};
  const float u = a.uniform[r];
  const double temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  const double top_p = a.top_ps ? a.top_ps[r] : a.top_p, min_p0 = a.min_ps ? a.min_ps[r] : a.min_p, min_p = min_p0 < 1.0 ? min_p0 : 1.0;  // the largest is always kept
  const int32_t top_k = temperature == 0 ? 1 : a.top_ks ? a.top_ks[r] : a.top_k;

  float m = -INFINITY;
  bool none = !(u >= 0.f && u <= 1.f) || !(temperature == 0 || (temperature >= 0x1p-63 && temperature < 0x1p64)) || top_p != top_p || min_p0 != min_p0;
  row.each([&](float x) {
    m = fmaxf(m, x);
    none |= x != x;
  });
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
    m = 0.f;
  }

  // Weights as whole numbers of 2^-shift.
  const int lg = 32 - __clz((a.vocab - 1) | 1), shift = 62 - lg < 46 ? 62 - lg : 46;
  const double inverse = 1.4426950408889634074 / (temperature == 0 ? 1.0 : temperature);
  auto weight = [&](float x) -> uint64_t {
    const double t = ((double)x - (double)m) * inverse;
    return t < -(double)(shift + 2) ? 0 : (uint64_t)__builtin_rint(exp2(t + shift));
  };

  auto clear = [&]() {
    for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
  };
  // Adds value(x) of the logits of keys low to high to bins by their key, the largest first.
  auto by_key = [&](uint32_t low, uint32_t high, int s, auto value) {
    row.each([&](float x) {
      const uint32_t k = key_of(x);
      if (k >= low && k <= high && x != -INFINITY) atomicAdd((unsigned long long*)&sh.bins[(high - k) >> s], (unsigned long long)value(x));
    });
  };
  // And to bins by their distance to the largest: 64 a unit of the logits over the temperature, the last one what is further away.
  const float per_unit = (float)(64.0 / (temperature == 0 ? 1.0 : temperature));
  auto bin_of = [&](float x) {
    const float d = (m - x) * per_unit;
    return d < (float)(kBins - 1) ? (uint32_t)d : (uint32_t)kBins - 1;
  };
  // The cut at which the values of the logits above the one `above` (keys greater than that), summed from the largest on, reach `target`.
  auto cut_at = [&](uint64_t target, uint32_t above, auto value) -> Cut {
    // sh.bins has the sums by distance
    find(sh, sh.bins, kBins, target);
    uint32_t bin = sh.found;
    uint64_t before = sh.found_before;
    if (bin == kBins) return Cut{above, 0, 0};  // all of them
    if (tid == 0) {
      sh.low = ~0u;
      sh.high = 0;
    }
    __syncthreads();
    uint32_t low = ~0u, high = 0;
    row.each([&](float x) {
      const uint32_t k = key_of(x);
      if (k > above && x != -INFINITY && bin_of(x) == bin) {
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
      by_key(low, high, s, value);
      __syncthreads();
      find(sh, sh.bins, kBins, target - before);
      if (sh.found >= kBins) break;  // (the sums are the ones that found the bin)
      before += sh.found_before;
      high = high - (sh.found << s);
      const uint32_t last = high - low < (1u << s) - 1 ? low : high - ((1u << s) - 1);
      low = last;
    }
    // `low` is the cut
    __syncthreads();
    if (tid == 0) sh.found = 0;
    __syncthreads();
    uint32_t n = 0;
    row.each([&](float x) { n += x != -INFINITY && key_of(x) == low; });
    if (n) atomicAdd(&sh.found, n);
    __syncthreads();
    const uint64_t one = value(of_key(low));
    const uint64_t equal = (target - before + one - 1) / one;
    return Cut{low, (uint32_t)(equal < sh.found ? equal : sh.found), sh.found};
  };

  Cut cut{0, 0, 0};
  if (top_k > 0 && (uint32_t)top_k < a.vocab) {
    clear();
    __syncthreads();
    row.each([&](float x) {
      if (x != -INFINITY) atomicAdd((unsigned long long*)&sh.bins[bin_of(x)], 1ull);
    });
    __syncthreads();
    cut = cut_at(top_k, 0, [](float) -> uint64_t { return 1; });
  }
  if (top_p < 1.0) {
    __syncthreads();
    clear();
    __syncthreads();
    row.each([&](float x) {
      if (x != -INFINITY && key_of(x) > cut.key) atomicAdd((unsigned long long*)&sh.bins[bin_of(x)], (unsigned long long)weight(x));
    });
    __syncthreads();
    uint64_t mine = 0;
    for (int i = tid; i < kBins; i += kThreads) mine += sh.bins[i];
    mine = wave_scan(mine);
    if (lane == 63) sh.wave_sum[wave] = mine;
    __syncthreads();
    uint64_t sum = 0;
    for (int i = 0; i < kWaves; ++i) sum += sh.wave_sum[i];
    __syncthreads();
    const uint64_t one = cut.equal ? weight(of_key(cut.key)) : 0, total = sum + cut.equal * one;
    const double share = __builtin_ceil(top_p * (double)total);
    const uint64_t target = share < 1.0 ? 1 : (uint64_t)share;
    if (target <= sum) {
      const Cut c = cut_at(target, cut.key, [&](float x) { return weight(x); });
      if (c.key > cut.key) cut = c;
    } else if (one) {
      const uint64_t equal = (target - sum + one - 1) / one;
      if (equal < cut.equal) cut.equal = (uint32_t)equal;
    }
  }

  // Which of the equal ones are kept: up to token `last`.
  uint32_t last = ~0u;
  const uint32_t pieces = row.slabs * kWaves;
  if (cut.equal < cut.there) {
    __syncthreads();
    for (uint32_t s = 0; s < row.slabs; ++s) {
      uint32_t n = 0;
      row.slab(s, [&](const float(&v)[PER], uint32_t) {
#pragma unroll
        for (int j = 0; j < PER; ++j) n += v[j] != -INFINITY && key_of(v[j]) == cut.key;
      });
      const uint64_t upto = wave_scan(n);
      if (lane == 63) sh.pieces[s * kWaves + wave] = upto;
    }
    __syncthreads();
    find(sh, sh.pieces, pieces, cut.equal);
    const uint32_t piece = sh.found;
    if (wave == piece % kWaves) {
      row.slab(piece / kWaves, [&](const float(&v)[PER], uint32_t at) {
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) n += v[j] != -INFINITY && key_of(v[j]) == cut.key;
        uint64_t before = sh.found_before + wave_scan(n) - n;
        if (before < cut.equal && before + n >= cut.equal)
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (v[j] != -INFINITY && key_of(v[j]) == cut.key && ++before == cut.equal) sh.token = at + j;
      });
    }
    __syncthreads();
    last = sh.token;
  }

  auto kept = [&](float x, uint32_t token) -> uint64_t {
    const uint32_t k = key_of(x);
    if (x == -INFINITY || k < cut.key || (k == cut.key && token > last)) return 0;
    const uint64_t w = weight(x);
    return min_p > 0.0 && exp2(((double)x - (double)m) * inverse) < min_p ? 0 : w;
  };
  __syncthreads();
  for (uint32_t s = 0; s < row.slabs; ++s) {
    uint64_t n = 0;
    row.slab(s, [&](const float(&v)[PER], uint32_t at) {
#pragma unroll
      for (int j = 0; j < PER; ++j) n += kept(v[j], at + j);
    });
    n = wave_scan(n);
    if (lane == 63) sh.pieces[s * kWaves + wave] = n;
  }
  __syncthreads();
  uint64_t sum = 0;
  for (uint32_t i = tid; i < pieces; i += kThreads) sum += sh.pieces[i];
  sum = wave_scan(sum);
  if (lane == 63) sh.wave_sum[wave] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < kWaves; ++i) sum += sh.wave_sum[i];
  __syncthreads();
  // the first token up to which the sum exceeds u of the whole: reaches the next whole number
  uint64_t target = (uint64_t)__builtin_floor((double)u * (double)sum) + 1;
  if (target > sum) target = sum;
  find(sh, sh.pieces, pieces, target);
  const uint32_t piece = sh.found;
  if (wave == piece % kWaves) {
    row.slab(piece / kWaves, [&](const float(&v)[PER], uint32_t at) {
      uint64_t w[PER], n = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) n += w[j] = kept(v[j], at + j);
      uint64_t before = sh.found_before + wave_scan(n) - n;
      if (before < target && before + n >= target)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (before < target && before + w[j] >= target) a.tokens[r] = at + j;
          before += w[j];
        }
    });
  }
}

}  // namespace

hipError_t launch_sample(int dtype, const SampleRows& a, hipStream_t st) {
  switch (dtype) {
    case 0: sample_kernel<TypeF32><<<a.nrows, kThreads, 0, st>>>(a); break;
    case 1: sample_kernel<TypeF16><<<a.nrows, kThreads, 0, st>>>(a); break;
    default: sample_kernel<TypeBF16><<<a.nrows, kThreads, 0, st>>>(a);
  }
  return hipGetLastError();
}

}  // namespace dz
