// Log probabilities and entropies straight from hidden states and the
// language-model head: the products are reduced to softmax statistics where
// they are made, and the logits are never stored.
#include "dz_lds.h"
#include "dz_token_loss.h"
#include "dz_token_math.h"

#include <type_traits>

namespace dz {
namespace {

// Products of M = 16 or 32 head rows by M tokens. A lane holds 16 bytes of a row's width: row l % M of
// the M, chunk l / M of the 64 / M that one step takes. The results: lane l holds token l % M, head rows
// 4 (l / M) .. + 3 of every 256 / M.
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <int M>
using Acc = std::conditional_t<M == 16, f32x4, f32x16>;

template <class T>
struct Frag;
template <>
struct Frag<TypeF16> {
  typedef TypeF16::V Loose __attribute__((aligned(2)));  // at any element
  using V = TypeF16::V;
  __device__ static f32x4 mma(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  __device__ static f32x16 mma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<TypeBF16> {
  typedef TypeBF16::V Loose __attribute__((aligned(2)));
  using V = TypeBF16::V;
  __device__ static f32x4 mma(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  __device__ static f32x16 mma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<TypeF32> {
  typedef TypeF32::V Loose __attribute__((aligned(4)));
  using V = TypeF32::V;
  // the chunks' columns in the order (0, 4, ...), (1, 5, ...), the same on both sides
  __device__ static f32x4 mma(V a, V b, f32x4 c) {
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  __device__ static f32x16 mma(V a, V b, f32x16 c) {
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

struct Work {
  uint32_t* count;   // live rows; NULL: every row is taken as one, in its order
  uint32_t* row_of;  // live row -> row
  uint32_t* live_of;  // row -> live row
  float* token_logit;  // per live row
  float4* partial;     // (live row, head tile)
};

__host__ __device__ inline uint64_t align256(uint64_t x) { return (x + 255) / 256 * 256; }
inline uint32_t head_tiles(uint32_t vocab, uint32_t tile) { return (vocab + tile - 1) / tile; }
inline Work work_of(void* p, uint32_t nrows) {
  const uint64_t n = align256((uint64_t)nrows * 4);
  char* c = (char*)p;
  return Work{(uint32_t*)c, (uint32_t*)(c + 256), (uint32_t*)(c + 256 + n), (float*)(c + 256 + 2 * n), (float4*)(c + 256 + 3 * n)};
}

// Numbers the rows that a token is asked for.
__global__ __launch_bounds__(1024) void live_rows_kernel(HeadRows a, Work w) {
  __shared__ uint32_t wave_live[16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  uint32_t base = 0;
  for (uint32_t r0 = 0; r0 < a.nrows; r0 += 1024) {
    const uint32_t r = r0 + tid;
    const bool live = r < a.nrows && a.tokens[r] != a.ignore;
    const uint64_t m = __ballot(live);
    __syncthreads();
    if (lane == 0) wave_live[wv] = (uint32_t)__popcll(m);
    __syncthreads();
    uint32_t before = base, all = base;
    for (uint32_t i = 0; i < 16; ++i) {
      if (i < wv) before += wave_live[i];
      all += wave_live[i];
    }
    if (live) {
      const uint32_t at = before + (uint32_t)__popcll(m & ((1ull << lane) - 1));
      w.row_of[at] = r;
      w.live_of[r] = at;
    }
    base = all;
  }
  if (tid == 0) *w.count = base;
}

// 16 bytes from column `col` of a row; columns past the width are 0. Rows start at any element.
template <class T>
__device__ __forceinline__ typename T::V load16(const typename T::Elem* row, uint32_t col, uint32_t width) {
  if (col + T::kPer16 <= width) return *(const typename Frag<T>::Loose*)(row + col);
  typename T::V v;
  for (int j = 0; j < T::kPer16; ++j) v[j] = col + j < width ? row[col + j] : (typename T::Elem)0.f;
  return v;
}

// f over the 64 / M lanes that hold the same token.
template <int M, class F>
__device__ __forceinline__ float over_lanes(float x, F f) {
  if (M == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// TF x M tokens' logits over a lane's head rows (those of VF products) to their statistics over the
// lanes that hold the same token. v0: the first head row of the wave. Leaves the logits of `tok`
// (2^32 - 1: none).
template <int M, int TF, int VF>
__device__ __forceinline__ void lane_stats(Acc<M> (&acc)[TF][VF], uint32_t v0, uint32_t vocab, const uint32_t (&tok)[TF],
                                           float* const (&token_logit)[TF], SoftStats (&st)[TF]) {
  const uint32_t lane = threadIdx.x & 63, first = v0 + 4 * (lane / M);
  auto row = [](int i, int j) { return (uint32_t)(i * M + j / 4 * (256 / M) + j % 4); };
  constexpr int N = M * M / 64;
  if (v0 + M * VF > vocab) {  // head rows past the last one take no part
#pragma unroll
    for (int n = 0; n < TF; ++n)
#pragma unroll
      for (int i = 0; i < VF; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (first + row(i, j) >= vocab) acc[n][i][j] = -INFINITY;
  }
#pragma unroll
  for (int n = 0; n < TF; ++n) {
    const uint32_t rel = tok[n] - first;
    if (__any(rel < M * VF)) {
      float x = 0.f;
      bool mine = false;
#pragma unroll
      for (int i = 0; i < VF; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (rel == row(i, j)) {
            x = acc[n][i][j];
            mine = true;
          }
      if (mine) *token_logit[n] = x;
    }
  }
#pragma unroll
  for (int n = 0; n < TF; ++n) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VF; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, acc[n][i][j]);
    st[n] = SoftStats::of(over_lanes<M>(m, [](float a, float b) { return fmaxf(a, b); }));
  }
#pragma unroll
  for (int n = 0; n < TF; ++n) {
    st[n].template add<true, VF * N>([&](int i) { return acc[n][i / N][i % N]; }, kLog2e);
    st[n].s = over_lanes<M>(st[n].s, [](float a, float b) { return a + b; });
    st[n].t = over_lanes<M>(st[n].t, [](float a, float b) { return a + b; });
  }
}

// A workgroup of WT x WV waves takes M TF WT live rows by M VF WV head rows, in slabs of 128
// bytes a row through LDS, STAGES of them: the next ones are on their way while this one's
// products run.
// What bounds it: up to 64 rows reading the head (64 rows by 50,272 tokens, 5,120 wide, fp16: 95 us, 5.4
// TB/s; one row 85 us, 6.0 TB/s), then the matrix units, under the power limit (2,048 rows, 2,560 wide, bf16: 498 us,
// 1.06 PFLOP/s, clocks at 2.0-2.1 GHz; a library's product of such a shape reaches 0.89).
//
// A slab's 16-byte chunk c of row r lies at r * 128 + (c ^ swizzle(r)) * 16.
__device__ __forceinline__ uint32_t swizzle(uint32_t r) { return (r >> 1) & 7; }
__device__ u32x4 zeros16[1];  // what the columns past the width are read from

// All but the last N of this wave's loads are done, and every wave of the workgroup is here.
template <int N>
__device__ __forceinline__ void arrive() {
  static_assert(N < 64, "a count of six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Every wave of the workgroup is here, and what it wrote to LDS is; loads on their way stay there.
__device__ __forceinline__ void arrive_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The row that is the at-th of the live ones, and its token (2^32 - 1: none that is asked for).
__device__ __forceinline__ uint32_t row_of(const Work& w, uint32_t at, uint32_t count) {
  if (at >= count) at = count - 1;
  return w.count ? w.row_of[at] : at;
}
__device__ __forceinline__ uint32_t token_of(const HeadRows& a, const Work& w, uint32_t at, uint32_t count) {
  const int64_t t = at < count ? a.tokens[row_of(w, at, count)] : -1;
  return t >= 0 && t < (int64_t)a.vocab ? (uint32_t)t : ~0u;
}

// The statistics of a tile whose logits are there, from all waves of the workgroup.
template <int M, int TF, int VF, int WT, int WV>
__device__ __forceinline__ void finish_tile(const HeadRows& a, const Work& w, Acc<M> (&acc)[TF][VF], const uint32_t (&tok)[TF],
                                            SoftStats (&sh)[WV][M * TF * WT], uint32_t vt, uint32_t mt, uint32_t count, uint32_t tiles) {
  constexpr uint32_t MT = M * TF * WT, NT = M * VF * WV;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wt = wave % WT, wv = wave / WT;
  float* token_logit[TF];
  SoftStats st[TF];
#pragma unroll
  for (int i = 0; i < TF; ++i) token_logit[i] = w.token_logit + mt * MT + (wt * TF + i) * M + lane % M;
  lane_stats<M>(acc, vt * NT + wv * M * VF, a.vocab, tok, token_logit, st);
  if (lane < M)
#pragma unroll
    for (int i = 0; i < TF; ++i) sh[wv][(wt * TF + i) * M + lane] = st[i];
  arrive_lds();
  for (uint32_t r = threadIdx.x; r < MT; r += 64 * WT * WV) {
    const uint32_t at = mt * MT + r;
    if (at >= count) break;
    SoftStats s = sh[0][r];
    for (int i = 1; i < WV; ++i) s.join(sh[i][r], kLog2e);
    w.partial[(uint64_t)at * tiles + vt] = float4{s.m, s.s, s.t, 0.f};
  }
}

template <class T, int M, int TF, int VF, int WT, int WV, int STAGES, bool ONCE, bool DIRECT>
__global__ __launch_bounds__(64 * WT * WV, M == 32 || STAGES == 5 ? 1 : 2) void head_tile_kernel(HeadRows a, Work w, uint32_t tiles) {
  using Elem = typename T::Elem;
  using V = typename T::V;
  constexpr uint32_t E = T::kPer16, K = 8 * E, WAVES = WT * WV;
  constexpr uint32_t MT = M * TF * WT, NT = M * VF * WV, ROWS = MT + NT, LOADS = ROWS / 8 / WAVES;
  static_assert(ROWS % (8 * WAVES) == 0, "loads");
  static_assert(STAGES >= 2 && (STAGES == 2 || DIRECT), "stages");
  __shared__ __attribute__((aligned(128))) char slots[STAGES][ROWS * 128];
  __shared__ SoftStats sh[WV][MT];
  const uint32_t count = w.count ? *w.count : a.nrows, mtiles = (count + MT - 1) / MT;
  // Workgroups go to the 8 XCDs in turn: an XCD takes every eighth of the head's tiles, and all
  // live rows of one after another, so that its L2 holds the tile's slabs for them. A workgroup takes
  // every gridDim / 8-th of its XCD's list.
  const uint32_t xcd = blockIdx.x % 8, stride = gridDim.x / 8;
  auto head_tile = [&](uint32_t n) { return n / mtiles * 8 + xcd; };
  auto there = [&](uint32_t n) { return head_tile(n) < tiles; };
  uint32_t tile = blockIdx.x / 8;
  if (!mtiles || !there(tile)) return;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wt = wave % WT, wv = wave / WT;
  // A load takes 8 rows of hidden states or of the head; this lane's row of load i, at its chunk.
  constexpr uint32_t HLOADS = MT / 8 / WAVES;
  static_assert(MT % (8 * WAVES) == 0, "a wave's load i is of the same kind for all waves");
  static_assert(WAVES % 2 == 0, "a lane's chunk is the same for all of its loads");
  const uint32_t chunk = (lane & 7) ^ swizzle(wave * 8 + (lane >> 3)), lane_row = wave * 8 + (lane >> 3);
  using Offset = std::conditional_t<DIRECT, uint32_t, uint64_t>;  // bytes; the launch looks after the 32 bits
  const char* const hidden0 = (const char*)a.hidden;
  const char* weight0;  // of the tile that is being loaded
  Offset from[LOADS];
  uint32_t rows[HLOADS];
  auto take_rows = [&](uint32_t n) {  // the rows of a tile, ahead of its loads
#pragma unroll
    for (uint32_t i = 0; i < HLOADS; ++i) rows[i] = row_of(w, n % mtiles * MT + i * WAVES * 8 + lane_row, count);
  };
  auto take_tile = [&](uint32_t n) {
    const uint32_t v0 = head_tile(n) * NT;
    weight0 = (const char*)a.weight + (int64_t)v0 * a.weight_stride * sizeof(Elem);
#pragma unroll
    for (uint32_t i = 0; i < LOADS; ++i) {
      const uint32_t v = (i - HLOADS) * WAVES * 8 + lane_row;
      const uint64_t at = i < HLOADS ? (uint64_t)rows[i < HLOADS ? i : 0] * a.hidden_stride : (uint64_t)(v0 + v < a.vocab ? v : a.vocab - 1 - v0) * a.weight_stride;
      from[i] = (Offset)(at * sizeof(Elem)) + chunk * 16;
    }
  };
  Acc<M> acc[TF][VF];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TF; ++i)
#pragma unroll
      for (int j = 0; j < VF; ++j) acc[i][j] = Acc<M>(0.f);
  };
  // Products of the slab in `here`, in groups of TF; `between` runs after each of the first half of the
  // groups. A group's operands are read while the two before it run.
  constexpr int PARTS = 8 * M / 64, GROUPS = PARTS * VF;
  uint32_t at[PARTS];  // this lane's chunks
#pragma unroll
  for (int n = 0; n < PARTS; ++n) at[n] = (lane % M) * 128 + ((n * (64 / M) + lane / M) ^ swizzle(lane % M)) * 16;
  auto products = [&](const char* here, auto between) {
    const char* bt = here + wt * M * TF * 128;
    const char* bv = here + (MT + wv * M * VF) * 128;
    V xt[PARTS][TF], xv[GROUPS];
    auto read_v = [&](int g) { xv[g] = *(const V*)(bv + g % VF * M * 128 + at[g / VF]); };
    auto read_t = [&](int n, int i) { xt[n][i] = *(const V*)(bt + i * M * 128 + at[n]); };
#pragma unroll
    for (int i = 0; i < TF; ++i) read_t(0, i);
    read_v(0);
    if (GROUPS > 1) read_v(1);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + 2 < GROUPS) read_v(g + 2);
#pragma unroll
      for (int i = 0; i < TF; ++i)
        if (g / VF + 1 < PARTS && g % VF == (VF - 1 - TF + i > 0 ? VF - 1 - TF + i : 0)) read_t(g / VF + 1, i);
#pragma unroll
      for (int i = 0; i < TF; ++i) acc[i][g % VF] = Frag<T>::mma(xv[g], xt[g / VF][i], acc[i][g % VF]);
      if (g < GROUPS / 2) between(g);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  uint32_t tok[TF];  // of the tile's rows, loaded when its products begin
  auto take_tokens = [&](uint32_t n) {
#pragma unroll
    for (int i = 0; i < TF; ++i) tok[i] = token_of(a, w, n % mtiles * MT + (wt * TF + i) * M + lane % M, count);
  };
  auto finish = [&](uint32_t n) { finish_tile<M, TF, VF, WT, WV>(a, w, acc, tok, sh, head_tile(n), n % mtiles, count, tiles); };

  const uint32_t slabs = (a.width + K - 1) / K;
  if constexpr (DIRECT) {
    // The slabs of all tiles follow each other without a stop: the first ones of a tile are on their way
    // while the last products of the tile before it run, and its statistics.
    const uint32_t full = a.width / K;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&slots[0][wave * 1024]);
    auto next_slot = [](uint32_t s) { return s + 1 == STAGES ? 0 : s + 1; };
    uint32_t load_tile = tile, load_k = 0, fill = 0;  // the next slab to load, and its place
    bool loading = true;
    auto load = [&](uint32_t i, uint32_t lds) {
      if (i < HLOADS) to_lds<false>(hidden0 + (uint64_t)load_k * 128, from[i], lds + i * WAVES * 1024);
      else to_lds<ONCE>(weight0 + (uint64_t)load_k * 128, from[i], lds + i * WAVES * 1024);
    };
    // a slab of which the last columns, or all, lie past the width
    auto load_end = [&](uint32_t lds) {
#pragma unroll
      for (uint32_t i = 0; i < LOADS; ++i) {
        const char* p = (i < HLOADS ? hidden0 : weight0) + from[i] + (uint64_t)load_k * 128;
        if (!loading || load_k * K + chunk * E >= a.width) p = (const char*)zeros16;
        to_lds(p, lds + i * WAVES * 1024);
      }
    };
    auto loaded = [&]() {
      fill = next_slot(fill);
      if (++load_k < slabs || !loading) return;
      load_k = 0;
      load_tile += stride;
      loading = there(load_tile);
      if (loading) {
        take_tile(load_tile);
        take_rows(load_tile + stride);
      }
    };
    take_rows(tile);
    take_tile(tile);
    take_rows(tile + stride);
    for (uint32_t k = 0; k < STAGES - 1; ++k) {
      load_end(lds0 + fill * ROWS * 128);
      loaded();
    }
    uint32_t slot = 0;
    for (; there(tile); tile += stride) {
      clear();
      take_tokens(tile);
      for (uint32_t k = 0; k < slabs; ++k) {
        arrive<(STAGES - 2) * LOADS>();  // slab k is there, and the products of slab k - 1, whose place the next one takes, are done
        const uint32_t lds = lds0 + fill * ROWS * 128;
        const bool whole = loading && load_k < full;
        // with more than two stages, slabs past the last one are loaded too (zeros), so that the wait is one number
        if (!whole && (STAGES > 2 || loading)) load_end(lds);
        products(slots[slot], [&](int g) {
#pragma unroll
          for (uint32_t i = 0; i < LOADS; ++i)
            if (i * (GROUPS / 2) / LOADS == (uint32_t)g && whole) load(i, lds);
        });
        loaded();
        slot = next_slot(slot);
      }
      finish(tile);
    }
    if (STAGES > 2) arrive<0>();  // a workgroup must not end, and give its LDS away, with loads to it on their way
  } else {
    u32x4 held[LOADS];  // a slab on its way
    auto fetch = [&](uint32_t k) {
      const bool tail = (k + 1) * K > a.width;
#pragma unroll
      for (uint32_t i = 0; i < LOADS; ++i) {
        const Elem* p = (const Elem*)((i < HLOADS ? hidden0 : weight0) + from[i] + (uint64_t)k * 128);
        const uint32_t at = k * K + chunk * E;
        const V x = tail ? load16<T>(p, 0, at < a.width ? a.width - at : 0) : (V)*(const typename Frag<T>::Loose*)p;
        held[i] = __builtin_bit_cast(u32x4, x);
      }
    };
    auto put = [&](char* there) {
#pragma unroll
      for (uint32_t i = 0; i < LOADS; ++i) *(u32x4*)(there + (wave + i * WAVES) * 1024 + lane * 16) = held[i];
    };
    for (; there(tile); tile += stride) {
      clear();
      take_tokens(tile);
      take_rows(tile);
      take_tile(tile);
      fetch(0);
      put(slots[0]);
      for (uint32_t k = 0; k < slabs; ++k) {
        __syncthreads();  // slab k is there; the products of slab k - 1 are done
        if (k + 1 < slabs) fetch(k + 1);
        products(slots[k & 1], [](int) {});
        if (k + 1 < slabs) put(slots[~k & 1]);
      }
      finish(tile);
    }
  }
}

// Many rows of fp32. The fp32 matrix instructions multiply at 1/16 of the rate of bf16's, so each
// number is taken as a sum of three bf16 numbers, hi + mid + lo, each the rounding of what the ones
// before leave: |mid| <= 2^-8 and |lo| <= 2^-17 of the number (bf16 has 8 bits, a rounding leaves half of the last one), and nothing is
// left of its 24 bits (of numbers below 2^-110 the last ones are below bf16's smallest number: 2^-120 keeps 14). A product is taken as the six of their nine products that can be above 2^-25 of it. What is left out, mid lo of
// both (2^-25 each, and close to it for 1 + 2^-8 - 2^-17) and lo lo (2^-34), is together not more than a rounding of an fp32 sum, 2^-24, which every
// product of the fp32 instructions has too. Against a kernel with fp32 instructions, by 50,272 tokens, 768
// wide: 2,048 rows 869 us for 1,230 (184 TFLOP/s of products of fp32 numbers, of 231 that six bf16 products at a library's rate
// would be), 300 rows, of whose 384 in tiles 84 are not there, 209 for 243. Taking apart is as much work for the vector units as the products
// are for the matrix units; 128 rows a tile share it (64: 1,066 us).
//
// An infinity among the operands (or a number that rounds to one) has no such sum: its parts make a
// NaN. A row of hidden states with one has no distribution whatever the head is; the logits of a head row with one are
// taken again by themselves.
//
// A workgroup of 2 x 4 waves takes 128 live rows by 256 head rows, in slabs of 32 columns, which come
// through registers: one slab is on its way, one is being taken apart into LDS, and one multiplies. A part's 16-byte chunk c
// of row r lies at r * 64 + (c ^ split_swizzle(r)) * 16.
__device__ __forceinline__ uint32_t split_swizzle(uint32_t r) {
  const uint32_t q = r >> 2 & 3;  // 0, 2, 3, 1: rows 0 to 3 and 12 to 15 of one chunk are read with rows 4 to 11 of the next
  return ((q ^ q >> 1) & 1) << 1 | q >> 1;
}
constexpr int kSplitTF = 4, kSplitVF = 4, kSplitWT = 2, kSplitWV = 4;
constexpr uint32_t kSplitGrid = 256;  // one workgroup a compute unit
constexpr uint32_t kSplitMT = 16 * kSplitTF * kSplitWT, kSplitNT = 16 * kSplitVF * kSplitWV;

__device__ __forceinline__ void take_apart(const float (&x)[8], bf16x8 (&part)[3]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[p][j] = (__bf16)r[j];
    const u32x4 bits = __builtin_bit_cast(u32x4, part[p]);
    if (p < 2)
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] -= __uint_as_float(j & 1 ? bits[j / 2] & 0xffff0000u : bits[j / 2] << 16);
  }
}

__global__ __launch_bounds__(512, 2) void head_split_kernel(HeadRows a, Work w, uint32_t tiles) {
  constexpr int TF = kSplitTF, VF = kSplitVF, WT = kSplitWT, WV = kSplitWV;
  constexpr uint32_t MT = kSplitMT, NT = kSplitNT, ROWS = MT + NT, UNITS = ROWS * 4, PER = (UNITS + 511) / 512;
  __shared__ __attribute__((aligned(256))) char slots[2][3][ROWS * 64];
  __shared__ SoftStats sh[WV][MT];
  __shared__ uint32_t bad[MT];  // rows with a number that is not finite
  const uint32_t count = w.count ? *w.count : a.nrows, mtiles = (count + MT - 1) / MT;
  // tiles in the order of head_tile_kernel
  uint32_t n = blockIdx.x / 8, vt, mt;
  if (!mtiles) return;
  for (; (vt = n / mtiles * 8 + blockIdx.x % 8) < tiles; n += gridDim.x / 8) {
    mt = n % mtiles;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave % WT, wv = wave / WT;
    if (tid < MT) bad[tid] = 0;

    // this thread's units of 8 columns: unit u is chunk u % 4 of row u / 4
    const float* from[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
      const uint32_t r = (i * 512 + tid) / 4 < ROWS ? (i * 512 + tid) / 4 : ROWS - 1;
      const uint32_t v = vt * NT + r - MT;
      from[i] = r < MT ? (const float*)a.hidden + (int64_t)row_of(w, mt * MT + r, count) * a.hidden_stride
                       : (const float*)a.weight + (int64_t)(v < a.vocab ? v : a.vocab - 1) * a.weight_stride;
      from[i] += tid % 4 * 8;
    }
    uint32_t tok[TF];
#pragma unroll
    for (int i = 0; i < TF; ++i) tok[i] = token_of(a, w, mt * MT + (wt * TF + i) * 16 + lane % 16, count);
    Acc<16> acc[TF][VF];
#pragma unroll
    for (int i = 0; i < TF; ++i)
#pragma unroll
      for (int j = 0; j < VF; ++j) acc[i][j] = Acc<16>(0.f);

    struct Slab {
      f32x4 x[PER][2];
    };
    Slab even, odd;
    auto fetch_whole = [&](Slab& s, uint32_t k) {
#pragma unroll
      for (uint32_t i = 0; i < PER; ++i)
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) s.x[i][n] = *(const Frag<TypeF32>::Loose*)(from[i] + (uint64_t)k * 32 + 4 * n);
    };
    auto fetch = [&](Slab& s, uint32_t k) {  // any slab
      if ((k + 1) * 32 <= a.width) return fetch_whole(s, k);
      const uint32_t at = k * 32 + tid % 4 * 8;
#pragma unroll
      for (uint32_t i = 0; i < PER; ++i)
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) s.x[i][n] = load16<TypeF32>(from[i] + (uint64_t)k * 32 + 4 * n, 0, at + 4 * n < a.width ? a.width - at - 4 * n : 0);
    };
    auto put = [&](const Slab& s, char (&there)[3][ROWS * 64], int i) {
      if (i * 512 + wave * 64 >= UNITS) return;
      const uint32_t r = (i * 512 + tid) / 4, to = r * 64 + ((tid & 3) ^ split_swizzle(r)) * 16;
      float x[8];
      bool finite = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = s.x[i][j / 4][j % 4];
        if (i * 512 + wave * 64 < MT * 4) finite &= fabsf(x[j]) < INFINITY;
      }
      if (!finite) bad[r] = 1;
      bf16x8 part[3];
      take_apart(x, part);
#pragma unroll
      for (int p = 0; p < 3; ++p) *(bf16x8*)(there[p] + to) = part[p];
    };
    const uint32_t at = (lane % 16) * 64 + ((lane / 16) ^ split_swizzle(lane % 16)) * 16;
    auto products = [&](const char (&here)[3][ROWS * 64], auto between) {
      bf16x8 t[3][TF], v[2][3];
      auto read_v = [&](int j) {
#pragma unroll
        for (int p = 0; p < 3; ++p) v[j & 1][p] = *(const bf16x8*)(here[p] + (MT + (wv * VF + j) * 16) * 64 + at);
      };
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int i = 0; i < TF; ++i) t[p][i] = *(const bf16x8*)(here[p] + (wt * TF + i) * 16 * 64 + at);
      read_v(0);
#pragma unroll
      for (int j = 0; j < VF; ++j) {
        if (j + 1 < VF) read_v(j + 1);
        constexpr int kPart[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};  // the small ones first
#pragma unroll
        for (int n = 0; n < 6; ++n)
#pragma unroll
          for (int i = 0; i < TF; ++i) acc[i][j] = Frag<TypeBF16>::mma(v[j & 1][kPart[n][0]], t[kPart[n][1]][i], acc[i][j]);
        between(j);
      }
    };
    const uint32_t slabs = (a.width + 31) / 32;
    __syncthreads();  // `bad` is cleared
    fetch(even, 0);
    if (slabs > 1) fetch(odd, 1);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) put(even, slots[0], i);
    // Slab k multiplies; slab k + 1, which `next` holds, is taken apart; slab k + 2 is asked for. The
    // steps whose slab k + 2 is a whole one have no branch at their loads, at which the compiler would wait.
    auto step = [&](uint32_t k, Slab& next, Slab& after, auto whole) {
      arrive_lds();
      if (whole) fetch_whole(after, k + 2);
      else if (k + 2 < slabs) fetch(after, k + 2);
      const bool more = whole || k + 1 < slabs;
      products(slots[k & 1], [&](int j) {
        if (more && j < (int)PER) put(next, slots[~k & 1], j);
      });
    };
    uint32_t k = 0;
    for (; k + 3 < a.width / 32; k += 2) {
      step(k, odd, even, std::true_type());
      step(k + 1, even, odd, std::true_type());
    }
    for (; k < slabs; k += 2) {
      step(k, odd, even, std::false_type());
      if (k + 1 < slabs) step(k + 1, even, odd, std::false_type());
    }

    // logits that infinities have spoilt
    bool spoilt = false;
#pragma unroll
    for (int i = 0; i < TF; ++i)
#pragma unroll
      for (int j = 0; j < VF; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) spoilt |= acc[i][j][e] != acc[i][j][e];
    if (__any(spoilt)) {
#pragma unroll 1
      for (int n = 0; n < TF * VF * 4; ++n) {
        const int ni = n / (VF * 4), nj = n / 4 % VF, ne = n % 4;
        float x = 0.f;
#pragma unroll
        for (int m = 0; m < TF * VF * 4; ++m)
          if (m == n) x = acc[m / (VF * 4)][m / 4 % VF][m % 4];
        const uint32_t r = (wt * TF + ni) * 16 + lane % 16, v = vt * NT + (wv * VF + nj) * 16 + 4 * (lane / 16) + ne;
        if (x != x && !bad[r] && v < a.vocab) {
          const float* h = (const float*)a.hidden + (int64_t)row_of(w, mt * MT + r, count) * a.hidden_stride;
          const float* e = (const float*)a.weight + (int64_t)v * a.weight_stride;
          x = 0.f;
          for (uint32_t c = 0; c < a.width; ++c) x = __builtin_fmaf(h[c], e[c], x);
        }
#pragma unroll
        for (int m = 0; m < TF * VF * 4; ++m)
          if (m == n) acc[m / (VF * 4)][m / 4 % VF][m % 4] = x;
      }
    }
    finish_tile<16, TF, VF, WT, WV>(a, w, acc, tok, sh, vt, mt, count, tiles);
    __syncthreads();
  }
}

// One wave joins a row's statistics over the head's tiles.
__global__ __launch_bounds__(64) void head_join_kernel(HeadRows a, Work w, uint32_t tiles) {
  const uint32_t r = blockIdx.x, lane = threadIdx.x;
  const int64_t tok = a.tokens[r];
  if (tok == a.ignore) {
    if (lane == 0) a.logprobs[r] = a.entropy[r] = 0.f;
    return;
  }
  const uint32_t at = w.count ? w.live_of[r] : r;
  SoftStats st = SoftStats::of(-INFINITY);
  for (uint32_t i = lane; i < tiles; i += 256) {  // four loads at a time
    float4 p[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) p[j] = i + 64 * j < tiles ? w.partial[(uint64_t)at * tiles + i + 64 * j] : float4{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      SoftStats o;
      o.m = p[j].x;
      o.s = p[j].y;
      o.t = p[j].z;
      st.join(o, kLog2e);
    }
  }
  for (int off = 32; off >= 1; off >>= 1) {
    SoftStats o;
    o.m = __shfl_xor(st.m, off, 64);
    o.s = __shfl_xor(st.s, off, 64);
    o.t = __shfl_xor(st.t, off, 64);
    st.join(o, kLog2e);
  }
  if (lane == 0) {
    const bool valid = st.valid(), inside = tok >= 0 && tok < (int64_t)a.vocab;
    const float log2s = log2_hw(st.s);
    a.logprobs[r] = valid && inside ? st.lnq(w.token_logit[at], kLog2e, 1.f) : NAN;
    a.entropy[r] = valid ? kLn2 * (log2s - st.t / st.s) : NAN;
  }
}

// A workgroup's rows and head rows. Up to 64 rows the head's bytes bound the kernel, from there on the
// products: large tiles then (256 x 256 read and write half of what 128 x 128 do). Where such tiles
// would leave half of the 256 compute units without one, smaller ones that more of them share, and that keep more
// slabs on their way, since the width is then walked through at the pace of a load (2,048 rows by
// 1,000 tokens, 5,120 wide, fp16: 111 us in 32 large tiles, 49 in 256 small ones; at 128 large ones they
// meet: 2,048 by 4,000, 1,024 wide 40 and 35 us, 700 by 16,000 in 189 tiles 38 and 42). Rounds of tiles are
// not weighed: 50,272 tokens make 197 of 256 head rows, which leaves 59 compute units without one for one tile of
// rows (256 rows of 5,120 fp16: 158 us), and 2.31 tiles each take three rounds (300 fp32 rows of 768: 187 us).
struct Plan {
  uint32_t row_tile, head_tile;
};
Plan plan_of(int dtype, uint32_t nrows, uint32_t vocab) {
  const uint32_t row_tile = nrows <= 32 ? 32 : nrows <= 64 ? 64 : nrows <= 128 ? 128 : 256;
  const bool few_tiles = (uint64_t)head_tiles(vocab, 256) * ((nrows + row_tile - 1) / row_tile) <= 128;
  if (nrows <= 64) return Plan{row_tile, few_tiles ? 64u : 256u};
  if (few_tiles) return Plan{64, 128};
  if (dtype == DZ_F32) return Plan{kSplitMT, kSplitNT};
  return Plan{row_tile, 256};
}

template <class T, int M, int TF, int VF, int WT, int WV, int STAGES, bool ONCE>
void tile(const HeadRows& a, const Work& w, uint32_t tiles, bool direct, hipStream_t st) {
  const uint64_t all = (uint64_t)((tiles + 7) / 8 * 8) * ((a.nrows + M * TF * WT - 1) / (M * TF * WT));
  constexpr uint32_t kLds = STAGES * (M * TF * WT + M * VF * WV) * 128 + WV * M * TF * WT * sizeof(SoftStats);
  constexpr uint32_t resident = 256 * (160 * 1024 / kLds < 8 / (WT * WV) ? 160 * 1024 / kLds : 8 / (WT * WV));  // two waves a SIMD
  const uint32_t grid = all < resident ? (uint32_t)all : resident;
  if (direct) head_tile_kernel<T, M, TF, VF, WT, WV, STAGES, ONCE, true><<<grid, 64 * WT * WV, 0, st>>>(a, w, tiles);
  else head_tile_kernel<T, M, TF, VF, WT, WV, 2, false, false><<<grid, 64 * WT * WV, 0, st>>>(a, w, tiles);
}
template <class T>
void products(const HeadRows& a, const Work& w, const Plan& p, uint32_t tiles, hipStream_t st) {
  // whole 16-byte chunks, at offsets of 32 bits, can go to LDS without a stop in registers
  const uint64_t es = sizeof(typename T::Elem);
  const bool direct = ((uint64_t)a.hidden | (uint64_t)a.weight | (uint64_t)a.hidden_stride * es | (uint64_t)a.weight_stride * es | a.width * es) % 16 == 0 &&
                      (uint64_t)a.hidden_stride * es * a.nrows < (1ull << 32) && (uint64_t)a.weight_stride * es * p.head_tile < (1ull << 32);
  if (a.nrows <= 32) {
    if (p.head_tile == 64) return tile<T, 16, 2, 1, 1, 4, 6, true>(a, w, tiles, direct, st);
    return tile<T, 32, 1, 2, 1, 4, 3, true>(a, w, tiles, direct, st);
  }
  if (a.nrows <= 64) {
    if (p.head_tile == 64) return tile<T, 16, 4, 1, 1, 4, 5, true>(a, w, tiles, direct, st);
    return tile<T, 32, 2, 2, 1, 4, 3, true>(a, w, tiles, direct, st);
  }
  if (p.head_tile == 128) return tile<T, 16, 2, 4, 2, 2, 3, false>(a, w, tiles, direct, st);
  if constexpr (sizeof(typename T::Elem) == 2) {
    if (p.row_tile == 128) return tile<T, 32, 2, 4, 2, 2, 3, true>(a, w, tiles, direct, st);
    return tile<T, 16, 4, 8, 4, 2, 2, false>(a, w, tiles, direct, st);
  } else {
    const uint64_t all = (uint64_t)((tiles + 7) / 8 * 8) * ((a.nrows + kSplitMT - 1) / kSplitMT);
    head_split_kernel<<<all < kSplitGrid ? (uint32_t)all : kSplitGrid, 512, 0, st>>>(a, w, tiles);
  }
}

}  // namespace

int64_t head_workspace(int dtype, uint32_t nrows, uint32_t width, uint32_t vocab) {
  (void)width;
  return (int64_t)(256 + 3 * align256((uint64_t)nrows * 4) + (uint64_t)nrows * head_tiles(vocab, plan_of(dtype, nrows, vocab).head_tile) * sizeof(float4));
}

hipError_t launch_head(int dtype, const HeadRows& a, void* workspace, hipStream_t st) {
  const Plan p = plan_of(dtype, a.nrows, a.vocab);
  Work w = work_of(workspace, a.nrows);
  const uint32_t tiles = head_tiles(a.vocab, p.head_tile);
  if (a.nrows <= p.row_tile) {  // one tile, whichever rows are asked for: all of them
    w.count = nullptr;
  } else {
    live_rows_kernel<<<1, 1024, 0, st>>>(a, w);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (dtype == DZ_F32) products<TypeF32>(a, w, p, tiles, st);
  else if (dtype == DZ_F16) products<TypeF16>(a, w, p, tiles, st);
  else products<TypeBF16>(a, w, p, tiles, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  head_join_kernel<<<a.nrows, 64, 0, st>>>(a, w, tiles);
  return hipGetLastError();
}

}  // namespace dz
