// Attention of sequences that share a prompt.
//
// o = sum_j w_j v_j / sum_j w_j, w_j = 2^(c q k_j - m), c = scale log2 e, over the keys j that a query sees: its group's
// prompt, and its own sequence's keys up to itself. One pass over the keys with a running maximum m and sum.
//
// A workgroup takes a tile of rows of one key head: the queries of all sequences of a group and of all query heads
// that share the key head, row (sequence * length + token) * shared + head. Its keys are the prompt's and then those of each
// sequence that the tile touches, in tiles of their own. The prompt is read once for all of the tile's rows; a sequence's own
// keys are scored against the whole tile and masked for the rows of others, which costs products that the
// matrix units have to spare: a tile of single tokens waits for its own keys from memory.
#include "dz_prefix.h"

#include <type_traits>

#include "dz_lds.h"
#include "dz_token_math.h"

namespace dz {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Products of 32 keys (or columns of values) by 32 queries over 16 of the width (or 16 keys). A lane holds 8
// elements of row l % 32; the results: lane l holds query l % 32 and rows 8 b + 4 (l / 32) + r (b, r < 4) in
// element 4 b + r. Which 8 of the 16 a lane holds does not matter as long as both operands agree: scores take 8 (l / 32) + j,
// and the products with values 8 (j / 4) + 4 (l / 32) + j % 4, which is where the scores lie already.
template <class T>
struct Op;
template <>
struct Op<TypeF16> {
  using Frag = f16x8;
  __device__ static f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  __device__ static u32x4 widen(u32x2 c, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], scale, true))};
  }
};
template <>
struct Op<TypeBF16> {
  using Frag = bf16x8;
  __device__ static f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  __device__ static u32x4 widen(u32x2 c, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, true))};
  }
};
template <>
struct Op<TypeF32> {
  using Frag = f32x8;
  __device__ static f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  __device__ static u32x4 widen(uint32_t c, float scale) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, scale, true);
    return u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
  }
};

// f of a lane's value and of the other half wave's, which holds the same query.
template <class F>
__device__ __forceinline__ float both_halves(float x, F f) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// Where a 16-byte chunk c of row r lies in a tile of CH chunks a row: chunk c ^ swizzle(r). Sixteen consecutive rows
// at one chunk (a read of keys), and four rows at four chunks (a read of values), then lie in different banks.
template <int CH>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  if (CH == 8) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
  if (CH == 10) return r >> 3 & 1;
  if (CH == 12 || CH == 20) return r >> 2 & 3;
  if (CH == 24) return r >> 1 & 7;
  return (r & 3) << 2 | (r >> 2 & 3);
}

// QS: sixteenths of the width, rounded up to 4, 5, 6 or 8.
template <class T, int QS, bool BY_KEYS>
struct Shape {
  static constexpr int kWide = std::is_same_v<T, TypeF32> ? 2 : 1;  // chunks of 8 elements
  static constexpr int CH = 2 * QS * kWide;                           // chunks of 16 bytes a row
  static constexpr int WAVES = BY_KEYS && kWide == 2 ? 2 : 4;
  static constexpr int KT = BY_KEYS || kWide == 2 ? 32 : 64;  // keys of a tile
  static constexpr int ROWS = BY_KEYS ? 32 : 32 * WAVES;      // most rows of a workgroup
  static constexpr int TILE = KT * CH * 16;                    // bytes of a tile's keys, or of its values
  static constexpr int LOADERS = BY_KEYS ? 1 : WAVES;            // waves that load a tile
  static constexpr int SLABS = BY_KEYS ? WAVES : 1;
  static constexpr int PV = (QS + 1) / 2;  // products of 32 columns of values
};

template <class T, int QS, bool BY_KEYS, bool BYTES, int THREADS = 64 * Shape<T, QS, BY_KEYS>::WAVES>
__global__ __launch_bounds__(THREADS, BY_KEYS ? 1 : 2) void attend_kernel(Attend a, AttendPlan plan, float* partial, float2* partial_ms) {
  using S = Shape<T, QS, BY_KEYS>;
  using Elem = typename T::Elem;
  using Frag = typename Op<T>::Frag;
  constexpr int CH = S::CH, KT = S::KT, NK = KT / 32;
  __shared__ __attribute__((aligned(256))) char lds[S::SLABS][2][2][S::TILE];
  __shared__ uint32_t ends[S::ROWS + 1];  // key tiles up to the end of a sequence's (first: of the prompt's)
  __shared__ float2 stats[BY_KEYS ? S::WAVES : 1][32];
  __shared__ uint32_t lims[S::ROWS];  // keys that are looked at of each sequence

  // Workgroups go to the 8 XCDs in turn: each XCD takes consecutive items, whose keys its L2 holds for them.
  const uint32_t items = (uint32_t)a.groups * a.kv_heads * plan.tiles * plan.splits, per = gridDim.x / 8;
  const uint32_t item = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (item >= items) return;
  const uint32_t split = item % plan.splits, gh = item / plan.splits / plan.tiles;
  const uint32_t tile = plan.tiles - 1 - item / plan.splits % plan.tiles;  // the longest first
  const uint32_t g = gh / a.kv_heads, hk = gh % a.kv_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const uint32_t shared = a.heads / a.kv_heads, seq_rows = (uint32_t)a.length * shared, all_rows = seq_rows * a.sequences;

  // The tile's rows, the sequences they belong to, and how far each looks.
  // (A tile covers whole sequences, or lies inside of one: plan.tile_rows is a multiple of a sequence's rows or tiles restart at each.)
  uint32_t row0, rows;
  if ((uint32_t)plan.tile_rows >= seq_rows) {
    row0 = tile * plan.tile_rows;
    rows = all_rows - row0 < (uint32_t)plan.tile_rows ? all_rows - row0 : plan.tile_rows;
  } else {
    const uint32_t per_seq = (seq_rows + plan.tile_rows - 1) / plan.tile_rows, n = tile / per_seq, r = tile % per_seq * plan.tile_rows;
    row0 = n * seq_rows + r;
    rows = seq_rows - r < (uint32_t)plan.tile_rows ? seq_rows - r : plan.tile_rows;
  }
  const uint32_t n0 = row0 / seq_rows, nseq = (row0 + rows - 1) / seq_rows - n0 + 1;
  auto limit_of = [&](uint32_t n, uint32_t t) {  // own keys that token t of sequence n sees
    const int64_t p = a.positions ? a.positions[(uint64_t)g * a.sequences + n] : a.slots - a.length;
    const int64_t l = p + t + 1;
    return (uint32_t)(l < 0 ? 0 : l > a.slots ? a.slots : l);
  };
  uint32_t prefix_limit = 0;
  if (a.prefix_slots) {
    const int32_t l = a.prefix_lengths ? a.prefix_lengths[g] : a.prefix_slots;
    prefix_limit = l < 0 ? 0 : l > a.prefix_slots ? a.prefix_slots : l;
  }
  prefix_limit = __builtin_amdgcn_readfirstlane(prefix_limit);
  if (tid < nseq) {
    const uint32_t n = n0 + tid, last = n == (row0 + rows - 1) / seq_rows ? (row0 + rows - 1) % seq_rows / shared : a.length - 1;
    lims[tid] = limit_of(n, last);
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t e = (prefix_limit + KT - 1) / KT;
    ends[0] = e;
    for (uint32_t i = 0; i < nseq; ++i) ends[i + 1] = e += (lims[i] + KT - 1) / KT;
  }
  __syncthreads();
  const uint32_t key_tiles = __builtin_amdgcn_readfirstlane(ends[nseq]);

  // This lane's query.
  const uint32_t lane_row = (BY_KEYS ? 0 : wave * 32) + (lane & 31);
  const bool live = lane_row < rows;
  const uint32_t row = row0 + (live ? lane_row : 0), n_row = row / seq_rows, t_row = row % seq_rows / shared, h_row = hk * shared + row % shared;
  const uint32_t own_limit = live ? limit_of(n_row, t_row) : 0;
  const int64_t q_at = (int64_t)g * a.q_s[0] + (int64_t)n_row * a.q_s[1] + (int64_t)h_row * a.q_s[2] + (int64_t)t_row * a.q_s[3];
  Frag qf[QS];
#pragma unroll
  for (int s = 0; s < QS; ++s) {
    const uint32_t col = 16 * s + 8 * half;
    qf[s] = Frag(Elem(0.f));
    if (live && col < (uint32_t)a.width) qf[s] = *(const Frag*)((const Elem*)a.q + q_at + col);
  }

  // Tiles of keys, in turn: `step` apart.
  const uint32_t first = BY_KEYS ? split * S::WAVES + wave : split, step = BY_KEYS ? plan.splits * S::WAVES : plan.splits;
  struct Part {
    uint32_t k0, limit, n;  // the tile's first key, its part's end, and the sequence (2^32 - 1: the prompt)
  };
  uint32_t at_seq = 0;  // the part that the last tile asked for lies in
  auto part_of = [&](uint32_t i) {
    while (i >= __builtin_amdgcn_readfirstlane(ends[at_seq])) ++at_seq;
    if (at_seq == 0) return Part{i * KT, prefix_limit, ~0u};
    return Part{(i - (uint32_t)__builtin_amdgcn_readfirstlane(ends[at_seq - 1])) * KT, (uint32_t)__builtin_amdgcn_readfirstlane(lims[at_seq - 1]), n0 + at_seq - 1};
  };

  char(*slab)[2][S::TILE] = lds[BY_KEYS ? wave : 0];
  const uint32_t loader = BY_KEYS ? 0 : wave;
  // A tile's loads, keys before values, 64 chunks each.
  constexpr int OF_KEYS = KT * CH / 64, LOADS = 2 * OF_KEYS / S::LOADERS;
  static_assert(KT * CH % 64 == 0 && 2 * OF_KEYS % S::LOADERS == 0, "loads");
  struct Store {  // of keys or of values, from the tile's first one on
    const char* at;
    int64_t stride;  // bytes
    const uint8_t* scale;
    int64_t scale_stride;
  };
  constexpr int SIZE = BYTES ? 1 : sizeof(Elem);
  auto store_of = [&](const Part& p, bool values) {
    const KeyValues& kv = p.n == ~0u ? a.prefix : a.own;
    const int64_t n = p.n == ~0u ? 0 : p.n;
    const int64_t(&s)[4] = values ? kv.v_s : kv.k_s;
    Store x;
    x.at = (const char*)(values ? kv.v : kv.k) + SIZE * ((int64_t)g * s[0] + n * s[1] + (int64_t)hk * s[2] + (int64_t)p.k0 * s[3]);
    x.stride = SIZE * s[3];
    if (BYTES) {
      const int64_t(&c)[4] = values ? kv.v_scale_s : kv.k_scale_s;
      x.scale = (values ? kv.v_scale : kv.k_scale) + ((int64_t)g * c[0] + n * c[1] + (int64_t)hk * c[2] + (int64_t)p.k0 * c[3]);
      x.scale_stride = c[3];
    }
    return x;
  };
  // Row and chunk of a lane's i-th load. Keys past the part's end are the last one again: their weights are 0, and what these
  // multiply is finite where the last key's values are. Chunks past the width are the row's first: finite where the row is,
  // and multiplied by 0 (keys) or not stored (values).
  constexpr int PER_CHUNK = 16 / sizeof(Elem);
  auto place = [&](int i, uint32_t last, uint32_t& r, uint32_t& c) {
    const uint32_t slot = (i * S::LOADERS + loader) % OF_KEYS * 64 + lane, row = slot / CH;
    c = (slot % CH) ^ swizzle<CH>(row);
    if (c * PER_CHUNK >= (uint32_t)a.width) c = 0;
    r = row < last ? row : last;
  };
  auto load_direct = [&](const Part& p, int stage) {
    const Store ks = store_of(p, false), vs = store_of(p, true);
    const uint32_t to0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&slab[stage][0][0]);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t j = i * S::LOADERS + loader;
      const bool values = j >= OF_KEYS;
      uint32_t r, c;
      place(i, p.limit - 1 - p.k0, r, c);
      to_lds<false>(values ? vs.at : ks.at, r * (uint32_t)(values ? vs.stride : ks.stride) + c * 16, to0 + j * 1024);
    }
  };
  // 8-bit codes go through registers, where each becomes an element times its row's power of two (exactly).
  using Code = std::conditional_t<PER_CHUNK == 8, u32x2, uint32_t>;
  struct Staged {
    Code code[LOADS];
    uint8_t scale[LOADS];
  };
  auto load_codes = [&](const Part& p, Staged& s) {
    const Store ks = store_of(p, false), vs = store_of(p, true);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const Store& x = i * S::LOADERS + loader >= OF_KEYS ? vs : ks;
      uint32_t r, c;
      place(i, p.limit - 1 - p.k0, r, c);
      s.code[i] = *(const Code*)(x.at + r * x.stride + c * PER_CHUNK);
      s.scale[i] = x.scale[r * x.scale_stride];
    }
  };
  auto put_codes = [&](const Staged& s, int stage) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *(u32x4*)(&slab[stage][0][0] + ((i * S::LOADERS + loader) * 64 + lane) * 16) = Op<T>::widen(s.code[i], __uint_as_float((uint32_t)s.scale[i] << 23));
  };

  f32x16 o[S::PV];
#pragma unroll
  for (int d = 0; d < S::PV; ++d) o[d] = f32x16(0.f);
  float m = -INFINITY, l = 0.f;  // l: of this lane's keys
  const float c = a.scale * kLog2e;

  auto products = [&](const Part& p, int stage) {
    const uint32_t limit = p.n == ~0u ? prefix_limit : p.n == n_row ? own_limit : 0;
    if (__all(limit <= p.k0)) return;  // none of the wave's rows
    const char* kt = slab[stage][0];
    const char* vt = slab[stage][1];
    f32x16 s[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      s[i] = f32x16(0.f);
      const uint32_t r = i * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < QS; ++q) {
        Frag kf;
        if constexpr (S::kWide == 1) {
          kf = *(const Frag*)(kt + r * CH * 16 + ((2 * q + half) ^ swizzle<CH>(r)) * 16);
        } else {
          const f32x4 lo = *(const f32x4*)(kt + r * CH * 16 + ((4 * q + 2 * half) ^ swizzle<CH>(r)) * 16);
          const f32x4 hi = *(const f32x4*)(kt + r * CH * 16 + ((4 * q + 2 * half + 1) ^ swizzle<CH>(r)) * 16);
          kf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        s[i] = Op<T>::mma(kf, qf[q], s[i]);
      }
    }
    if (!__all(limit >= p.k0 + KT)) {
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (p.k0 + i * 32 + 8 * (j / 4) + 4 * half + j % 4 >= limit) s[i][j] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, s[i][j]);
    top = both_halves(top, [](float x, float y) { return fmaxf(x, y); }) * c;
    if (__any(top > m)) {
      const float m2 = fmaxf(m, top);
      const float f = m2 == -INFINITY ? 1.f : exp2_hw(m - m2);
      m = m2;
      l *= f;
#pragma unroll
      for (int d = 0; d < S::PV; ++d) o[d] *= f;
    }
    const float mm = m == -INFINITY ? 0.f : m;
    Frag w[NK][2];
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float e = exp2_hw(__builtin_fmaf(s[i][j], c, -mm));
        l += e;
        w[i][j / 8][j % 8] = (Elem)e;
      }
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          Frag vf;
          if constexpr (S::kWide == 1) {
            // four rows of 16 columns for each 16 lanes, which get a column each
            const uint32_t col = 32 * d + (lane & 31) / 16 * 16, group = col / 8 < CH ? col / 8 : CH - 2, chunk = group + (lane & 3) / 2;
            s16x4 part[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t r = i * 32 + k * 16 + j * 8 + 4 * half + (lane & 15) / 4;
              part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + r * CH * 16 + (chunk ^ swizzle<CH>(r)) * 16 + (lane & 1) * 8));
            }
            vf = __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
          } else {
            const uint32_t col = 32 * d + (lane & 31), chunk = col / 4 < CH ? col / 4 : CH - 1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t r = i * 32 + k * 16 + j / 4 * 8 + 4 * half + j % 4;
              vf[j] = *(const float*)(vt + r * CH * 16 + (chunk ^ swizzle<CH>(r)) * 16 + (lane & 3) * 4);
            }
          }
          o[d] = Op<T>::mma(vf, w[i][k], o[d]);
        }
  };

  // Two tiles' room: the next one is on its way while this one's products run.
  auto arrive_all = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // no load or read of LDS is left open
    if (!BY_KEYS) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (first < key_tiles) {
    Part now = part_of(first);
    Staged st;
    if constexpr (BYTES) {
      load_codes(now, st);
      put_codes(st, 0);
    } else {
      load_direct(now, 0);
    }
    int stage = 0;
    for (uint32_t i = first; i < key_tiles; i += step) {
      const bool more = i + step < key_tiles;
      Part next = now;
      if (more) next = part_of(i + step);
      arrive_all();
      if (more) {
        if constexpr (BYTES) load_codes(next, st);
        else load_direct(next, stage ^ 1);
      }
      products(now, stage);
      if constexpr (BYTES)
        if (more) put_codes(st, stage ^ 1);
      stage ^= 1;
      now = next;
    }
  }
  l = both_halves(l, [](float x, float y) { return x + y; });

  if constexpr (BY_KEYS) {
    // The waves' sums against the largest of their maxima.
    if (half == 0) stats[wave][lane] = float2{m, l};
    __syncthreads();  // every wave is through with its slab, too
    float top = -INFINITY;
    for (int i = 0; i < S::WAVES; ++i) top = fmaxf(top, stats[i][lane & 31].x);
    const float f = m == -INFINITY ? 0.f : exp2_hw(m - top);
    float sum = 0.f;
    for (int i = 0; i < S::WAVES; ++i) {
      const float2 x = stats[i][lane & 31];
      if (x.x != -INFINITY) sum += x.y * exp2_hw(x.x - top);
    }
    m = top;
    l = sum;
    constexpr int PITCH = S::PV * 32 + 4;  // floats of a row
    float* mine = (float*)lds + wave * 32 * PITCH;
    static_assert(S::WAVES * 32 * PITCH * 4 <= (int)sizeof(lds), "room");
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *(f32x4*)(mine + (lane & 31) * PITCH + 32 * d + 8 * b + 4 * half) =
            f32x4{o[d][4 * b] * f, o[d][4 * b + 1] * f, o[d][4 * b + 2] * f, o[d][4 * b + 3] * f};
    __syncthreads();
    if (wave != 0) return;  // (the sums that are left take one wave)
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f32x4 x = f32x4(0.f);
        for (int i = 0; i < S::WAVES; ++i) x += *(const f32x4*)((float*)lds + (i * 32 + (lane & 31)) * PITCH + 32 * d + 8 * b + 4 * half);
        for (int r = 0; r < 4; ++r) o[d][4 * b + r] = x[r];
      }
  }
  if (!live) return;
  if (plan.splits > 1) {
    const uint64_t at = ((uint64_t)gh * all_rows + row) * plan.splits + split;
    if (half == 0) partial_ms[at] = float2{m, l};
    float* to = partial + at * a.width;
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t col = 32 * d + 8 * b + 4 * half;
        if (col < (uint32_t)a.width) *(f32x4*)(to + col) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
      }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  Elem* to = (Elem*)a.out + (int64_t)g * a.out_s[0] + (int64_t)n_row * a.out_s[1] + (int64_t)h_row * a.out_s[2] + (int64_t)t_row * a.out_s[3];
  typedef Elem Quad __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < S::PV; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t col = 32 * d + 8 * b + 4 * half;
      if (col < (uint32_t)a.width)
        *(Quad*)(to + col) = Quad{(Elem)(o[d][4 * b] * inv), (Elem)(o[d][4 * b + 1] * inv), (Elem)(o[d][4 * b + 2] * inv), (Elem)(o[d][4 * b + 3] * inv)};
    }
}

// The splits' sums of each row, joined. 32 lanes a row, four columns a lane.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(Attend a, AttendPlan plan, const float* partial, const float2* partial_ms) {
  using Elem = typename T::Elem;
  const uint32_t shared = a.heads / a.kv_heads, seq_rows = (uint32_t)a.length * shared, all_rows = seq_rows * a.sequences;
  const uint64_t at = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32, total = (uint64_t)a.groups * a.kv_heads * all_rows;
  const uint32_t col = threadIdx.x % 32 * 4;
  if (at >= total || col >= (uint32_t)a.width) return;
  float m = -INFINITY;
  for (int i = 0; i < plan.splits; ++i) m = fmaxf(m, partial_ms[at * plan.splits + i].x);
  float l = 0.f;
  f32x4 o = f32x4(0.f);
  for (int i = 0; i < plan.splits; ++i) {
    const float2 ms = partial_ms[at * plan.splits + i];
    if (ms.x == -INFINITY) continue;  // saw no key
    const float f = exp2_hw(ms.x - m);
    l = __builtin_fmaf(ms.y, f, l);
    o += *(const f32x4*)(partial + (at * plan.splits + i) * a.width + col) * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const uint32_t gh = (uint32_t)(at / all_rows), row = (uint32_t)(at % all_rows), g = gh / a.kv_heads, h = gh % a.kv_heads * shared + row % shared;
  typedef Elem Quad __attribute__((ext_vector_type(4)));
  *(Quad*)((Elem*)a.out + (int64_t)g * a.out_s[0] + (int64_t)(row / seq_rows) * a.out_s[1] + (int64_t)h * a.out_s[2] +
           (int64_t)(row % seq_rows / shared) * a.out_s[3] + col) = Quad{(Elem)(o[0] * inv), (Elem)(o[1] * inv), (Elem)(o[2] * inv), (Elem)(o[3] * inv)};
}

template <class T, int QS, bool BY_KEYS>
void launch_one(const Attend& a, const AttendPlan& p, uint32_t grid, float* partial, float2* ms, hipStream_t st) {
  if (a.bytes) attend_kernel<T, QS, BY_KEYS, true><<<grid, 64 * Shape<T, QS, BY_KEYS>::WAVES, 0, st>>>(a, p, partial, ms);
  else attend_kernel<T, QS, BY_KEYS, false><<<grid, 64 * Shape<T, QS, BY_KEYS>::WAVES, 0, st>>>(a, p, partial, ms);
}
template <class T, int QS>
void launch_qs(const Attend& a, const AttendPlan& p, uint32_t grid, float* partial, float2* ms, hipStream_t st) {
  if (p.by_keys) launch_one<T, QS, true>(a, p, grid, partial, ms, st);
  else launch_one<T, QS, false>(a, p, grid, partial, ms, st);
}
template <class T>
hipError_t launch_typed(const Attend& a, const AttendPlan& p, void* workspace, hipStream_t st) {
  const uint64_t rows = (uint64_t)a.groups * a.heads * a.sequences * a.length;
  float2* ms = (float2*)workspace;
  float* partial = (float*)((char*)workspace + (rows * p.splits * 8 + 15) / 16 * 16);
  const uint64_t items = (uint64_t)a.groups * a.kv_heads * p.tiles * p.splits;
  const uint32_t grid = (uint32_t)((items + 7) / 8 * 8);
  const int qs = (a.width + 15) / 16;
  if (qs <= 4) launch_qs<T, 4>(a, p, grid, partial, ms, st);
  else if (qs == 5) launch_qs<T, 5>(a, p, grid, partial, ms, st);
  else if (qs == 6) launch_qs<T, 6>(a, p, grid, partial, ms, st);
  else launch_qs<T, 8>(a, p, grid, partial, ms, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  join_kernel<T><<<(uint32_t)((rows + 7) / 8), 256, 0, st>>>(a, p, partial, ms);
  return hipGetLastError();
}

}  // namespace

AttendPlan attend_plan(int dtype, const Attend& a) {
  const int64_t shared = a.heads / a.kv_heads, seq_rows = a.length * shared, heads = (int64_t)a.groups * a.kv_heads;
  AttendPlan p{};
  p.by_keys = seq_rows <= 32;
  const int64_t most = p.by_keys ? 32 : 128;
  if (seq_rows <= most) {
    p.tile_rows = (int32_t)(most / seq_rows * seq_rows);
    if (p.tile_rows > seq_rows * a.sequences) p.tile_rows = (int32_t)(seq_rows * a.sequences);
    p.tiles = (int32_t)((seq_rows * a.sequences + p.tile_rows - 1) / p.tile_rows);
  } else {
    p.tile_rows = (int32_t)most;
    p.tiles = (int32_t)((seq_rows + most - 1) / most * a.sequences);
  }
  // keys that a tile looks at, at most; a split takes 512 of them or more
  const int64_t seqs = p.tile_rows > seq_rows ? p.tile_rows / seq_rows : 1, keys = a.prefix_slots + seqs * a.slots;
  const int64_t want = (2 * 256 + heads * p.tiles - 1) / (heads * p.tiles), cap = keys / 512;
  p.splits = (int32_t)(want < cap ? want : cap);
  if (p.splits < 1) p.splits = 1;
  return p;
}

int64_t attend_workspace(const Attend& a, const AttendPlan& p) {
  if (p.splits == 1) return 0;
  const int64_t rows = (int64_t)a.groups * a.heads * a.sequences * a.length;
  return (rows * p.splits * 8 + 15) / 16 * 16 + rows * p.splits * a.width * 4;
}

hipError_t launch_attend(int dtype, const Attend& a, const AttendPlan& p, void* workspace, hipStream_t st) {
  switch (dtype) {
    case 0: return launch_typed<TypeF32>(a, p, workspace, st);
    case 1: return launch_typed<TypeF16>(a, p, workspace, st);
    default: return launch_typed<TypeBF16>(a, p, workspace, st);
  }
}

}  // namespace dz
