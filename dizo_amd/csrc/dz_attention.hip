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
//
// What bounds it, and what it measured (one MI355X; the floor: bytes at a large copy's 4.96 TB/s, or products at a large
// library product's 1,358 TFLOP/s in bf16):
//   single tokens   their keys from memory: 64 answers of up to 256 tokens after 2,048 keys, 40 heads of 128, 295 MB, 53 us (5.5 TB/s) and 6
//                   to join; floor 60
//   the same, 8 bit conversions next to the loads: 2 x 32 answers after 6,000, 8 key heads of 32, 28 us and 6 to join; floor 15
//   candidates      the way through one workgroup (lengths, then keys, scores, values, the waves' sums): 14 us; floor 8
//   prompts         one causal sequence of 4,096, 40 heads of 128: 220 us, 780 TFLOP/s; the products alone reach 1,030 under the power limit
//                   in this order (scores, weights, values by one wave)
// A lane holds one query: scores are taken as K Q^T and results as V^T P^T, so that maxima, sums and weights stay in the
// lane (two lanes a query) and weights are the second product's operand as they are. Values are read from LDS transposed.
#include "dz_attention.h"
#include "dz_lds.h"

namespace dz {
namespace {

// What a tile in LDS is.
enum Store {
  kOperands,   // elements, loaded straight to LDS
  kConverted,  // elements that were codes: loaded to registers and converted once for all waves
  kCodes,      // codes, loaded straight to LDS and converted by the wave that takes keys for itself; widths of whole chunks (32 single tokens
               // after 6,000 keys: 30 us, through registers 37; waves that share keys would convert each code four times)
};

// What an e8m0 scale stands for: 2^(s - 127), 0 being fp32's subnormal one, and NaN for 255. (The conversions of codes take s << 23 for that.)
__device__ __forceinline__ float power_of(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
}

// A row by itself, key by key: a lane takes a key's score, and then a column or two of the values. For rows whose sums are not finite:
// a product with a weight of 0 is NaN where the value is infinite or NaN, so that one such value reaches all rows that its tile was
// scored against, and sums of values near fp32's limits may leave it where their mean does not. Here a row meets the keys that it
// sees and no others, and o is the mean of the values so far.
template <class T, bool BYTES>
struct LoneRow {
  using Elem = typename T::Elem;
  const Elem* q;
  float o[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
  uint32_t lane = threadIdx.x & 63;

  __device__ static float value(const void* x, const uint8_t* power, int64_t at, int64_t power_at) {
    if constexpr (BYTES) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)x)[at], 0) * power_of(power[power_at]);
    return (float)((const Elem*)x)[at];
  }
  // Keys k0 ... k1 - 1, 64 at most; true when the answer is NaN whatever follows.
  __device__ bool keys(const Attend& a, const KeyValues& kv, uint32_t g, uint32_t n, uint32_t hk, uint32_t k0, uint32_t k1) {
    auto from = [&](const int64_t* s, uint32_t key) { return (int64_t)g * s[0] + (int64_t)n * s[1] + (int64_t)hk * s[2] + (int64_t)key * s[3]; };
    float s = -INFINITY;
    if (k0 + lane < k1) {
      const int64_t at = from(kv.k_s, k0 + lane), power_at = BYTES ? from(kv.k_scale_s, k0 + lane) : 0;
      s = 0.f;
#pragma unroll 1
      for (int i = 0; i < a.width; ++i) s = __builtin_fmaf((float)q[i], value(kv.k, kv.k_scale, at + i, power_at), s);
      s *= a.scale * kLog2e;
    }
    if (__any(s != s || s == INFINITY)) {
      o[0] = o[1] = NAN;
      m = 0.f;
      l = 1.f;
      return true;
    }
    float top = s;
    for (int d = 32; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
    top = fmaxf(top, m);
    const float e = s == -INFINITY ? 0.f : exp2_hw(s - top);
    float sum = e;
    for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
    const float before = l == 0.f ? 0.f : l * exp2_hw(m - top);
    m = top;
    l = before + sum;
    const float part = l == 0.f ? 0.f : 1.f / l;
    o[0] *= before * part;
    o[1] *= before * part;
#pragma unroll 1
    for (uint32_t key = k0; key < k1; ++key) {
      const float w = __shfl(e, key - k0) * part;
      const int64_t at = from(kv.v_s, key), power_at = BYTES ? from(kv.v_scale_s, key) : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < (uint32_t)a.width) o[i] = __builtin_fmaf(w, value(kv.v, kv.v_scale, at + lane + 64 * i, power_at), o[i]);
    }
    return false;
  }
};

// What a kernel is launched with.
struct Call {
  Attend a;
  AttendPlan plan;
  float* partial;  // sums of rows whose keys several workgroups take, and their maxima and sums of weights
  float2* partial_ms;
};

// Own keys that token t of sequence n sees.
__device__ __forceinline__ uint32_t own_keys(const Attend& a, uint32_t g, uint32_t n, uint32_t t) {
  const int64_t p = a.positions ? a.positions[(uint64_t)g * a.sequences + n] : a.slots - a.length;
  const int64_t l = p + t + 1;
  return (uint32_t)(l < 0 ? 0 : l > a.slots ? a.slots : l);
}
// Keys of the group's prompt.
__device__ __forceinline__ uint32_t prefix_keys(const Attend& a, uint32_t g) {
  if (!a.prefix_slots) return 0;
  const int32_t l = a.prefix_lengths ? a.prefix_lengths[g] : a.prefix_slots;
  return l < 0 ? 0 : l > a.prefix_slots ? a.prefix_slots : l;
}

// The rows first + (each set bit) of the workgroup's tile by themselves, one after another. Where they are and what they see
// is found again from the arguments: kept until here, it would take registers from the kernel's loop (8-bit answers: 36 us
// against 34).
template <class T, bool BY_KEYS, bool BYTES, uint32_t KT, uint32_t WAVES>
__device__ __forceinline__ void lone_rows(uint32_t first, uint32_t set) {
  using Elem = typename T::Elem;
  auto arguments = (const __attribute__((address_space(4))) Call*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(arguments));
  const Call& call = *(const Call*)arguments;
  const Attend& a = call.a;
  const AttendPlan& plan = call.plan;
  Item item;
  if (!item_of(a, plan, item)) return;
  const uint32_t lane = threadIdx.x & 63, g = item.g, shared = a.heads / a.kv_heads, seq_rows = (uint32_t)a.length * shared;
  const uint32_t row0 = tile_rows_of(plan, item.tile, seq_rows, seq_rows * a.sequences).row0, n0 = row0 / seq_rows;
  const uint32_t prefix_limit = __builtin_amdgcn_readfirstlane(prefix_keys(a, g)), prefix_tiles = (prefix_limit + KT - 1) / KT;
  auto mine = [&](uint32_t tile) { return (BY_KEYS ? tile / WAVES : tile) % item.splits == item.split; };
#pragma unroll 1
  for (; set; set &= set - 1) {
    const uint32_t lane_row = first + __builtin_ctz(set), row = row0 + lane_row;
    const uint32_t n = row / seq_rows, t = row % seq_rows / shared, h = item.hk * shared + row % shared, limit = own_keys(a, g, n, t);
    LoneRow<T, BYTES> x{(const Elem*)a.q + (int64_t)g * a.q_s[0] + (int64_t)n * a.q_s[1] + (int64_t)h * a.q_s[2] + (int64_t)t * a.q_s[3]};
    uint32_t begin = prefix_tiles;  // its own tiles' place among the workgroup's
    for (uint32_t i = n0; i < n; ++i) begin += (own_keys(a, g, i, a.length - 1) + KT - 1) / KT;
    bool done = false;
#pragma unroll 1
    for (uint32_t i = 0; i < prefix_tiles && !done; ++i)
      if (mine(i)) done = x.keys(a, a.prefix, g, 0, item.hk, i * KT, min((i + 1) * KT, prefix_limit));
#pragma unroll 1
    for (uint32_t i = 0; i * KT < limit && !done; ++i)
      if (mine(begin + i)) done = x.keys(a, a.own, g, n, item.hk, i * KT, min((i + 1) * KT, limit));
    const uint64_t to_row = item.splits > 1 ? partial_row(plan, item, lane_row) : 0;
    // (a mean: a sum of weights of 1 relative to 2^m of them all)
    if (item.splits > 1 && lane == 0) call.partial_ms[to_row] = x.l == 0.f ? float2{-INFINITY, 0.f} : float2{x.m + log2_hw(x.l), 1.f};
    Elem* to = (Elem*)a.out + (int64_t)g * a.out_s[0] + (int64_t)n * a.out_s[1] + (int64_t)h * a.out_s[2] + (int64_t)t * a.out_s[3];
    for (int i = 0; i < 2; ++i) {
      const uint32_t col = lane + 64 * i;
      if (col >= (uint32_t)a.width) continue;
      if (item.splits > 1) call.partial[to_row * a.width + col] = x.o[i];
      else to[col] = (Elem)(prefix_limit + limit == 0 ? 0.f : x.l == 0.f ? NAN : x.o[i]);
    }
  }
}

// QS: sixteenths of the width, rounded up to 4, 5, 6 or 8. BY_KEYS: WAVES waves take keys for themselves; otherwise four share them.
template <class T, int QS, bool BY_KEYS, Store STORE, int OF_WAVES>
struct Shape {
  static constexpr bool kWide = std::is_same_v<T, TypeF32>;
  static constexpr int CH = STORE == kCodes ? QS : kWide ? 4 * QS : 2 * QS;  // chunks of 16 bytes a row
  static constexpr int STEPS = STORE == kCodes ? (QS + 1) / 2 * 2 : QS;        // products along the width
  static constexpr int WAVES = OF_WAVES;
  static_assert(BY_KEYS || WAVES == 4, "shared tiles");
  static constexpr int KT = BY_KEYS || kWide ? 32 : 64;    // keys of a tile
  static constexpr int ROWS = BY_KEYS ? 32 : 32 * WAVES;  // most rows of a workgroup
  static constexpr int TILE = KT * CH * 16;                // bytes of a tile's keys, or of its values
  static constexpr int LOADERS = BY_KEYS ? 1 : WAVES;        // waves that load a tile
  static constexpr int SLABS = BY_KEYS ? WAVES : 1;
  static constexpr int PV = (QS + 1) / 2;  // products of 32 columns of values
  // Tiles in LDS. Waves that take keys for themselves have one each: the other waves' loads are on their way meanwhile, and
  // twice as many of them find room (candidates fp16 by four waves: 20 us, with two tiles 28).
  static constexpr int STAGES = BY_KEYS && STORE != kCodes ? 1 : 2;
  // workgroups that a compute unit's LDS and registers hold: eight waves, or four with more than half of the LDS
  static constexpr int RESIDENT = (4 * SLABS / WAVES * STAGES * 2 * TILE > 72 * 1024 ? 4 : 8) / WAVES;
};

template <class T, int QS, bool BY_KEYS, Store STORE, int OF_WAVES, int THREADS = 64 * OF_WAVES,
          int RESIDENT = Shape<T, QS, BY_KEYS, STORE, OF_WAVES>::RESIDENT>
__global__ __launch_bounds__(THREADS, (THREADS * RESIDENT + 255) / 256) void attend_kernel(Call call) {
  const Attend& a = call.a;
  const AttendPlan& plan = call.plan;
  using S = Shape<T, QS, BY_KEYS, STORE, OF_WAVES>;
  using Elem = typename T::Elem;
  using Frag = typename Op<T>::Frag;
  // Weights of codes carry their row's power of two, which may leave the range of fp16: those are bf16 (and codes are bf16 numbers), for
  // fp16 results two of them, the nearest one and the nearest to what that leaves: 2^-16 of a weight at most.
  using TV = std::conditional_t<STORE == kCodes && std::is_same_v<T, TypeF16>, TypeBF16, T>;
  using FragV = typename Op<TV>::Frag;
  // Weights are 2^(s + kBias - m), where m trails the row's largest score by kLag at most: sums change their scale a few times, and not
  // with each tile. fp16 weights are taken up to 2^15 that way, so that they have all of their bits down to 2^-25 of the row's largest, and
  // what rounds to 0 is below 2^-36 of it: 2^24 keys of that lose 2^-12 (with the largest at 1, 2^20 keys of 2^-26 would be lost
  // whole, 1.6 % of the result). bf16 has fp32's range.
  constexpr bool kHalf = std::is_same_v<TV, TypeF16>, kTwo = std::is_same_v<T, TypeF16> && !kHalf;
  // Those of codes times powers of two are taken 2^16 higher, to have bits left at 2^-127, the least power there is.
  constexpr float kBias = kHalf ? 11.f : STORE == kCodes ? 16.f : 0.f, kLag = kHalf ? 4.f : 8.f;
  constexpr int CH = S::CH, KT = S::KT, NK = KT / 32;
  constexpr bool BYTES = STORE != kOperands;
  __shared__ __attribute__((aligned(256))) char lds[S::SLABS][S::STAGES][2][S::TILE];
  __shared__ float2 stats[BY_KEYS ? S::WAVES : 1][32];
  __shared__ __attribute__((aligned(16))) float powers[STORE == kCodes ? S::WAVES : 1][32];  // of a tile's values

  Item item;
  if (!item_of(a, plan, item)) return;
  const uint32_t g = item.g, hk = item.hk, split = item.split, splits = item.splits;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const uint32_t shared = a.heads / a.kv_heads, seq_rows = (uint32_t)a.length * shared, all_rows = seq_rows * a.sequences;

  // The tile's rows, the sequences they belong to, and how far each looks.
  // (A tile covers whole sequences, or lies inside of one: plan.tile_rows is a multiple of a sequence's rows or tiles restart at each.)
  const TileRows tr = tile_rows_of(plan, item.tile, seq_rows, all_rows);
  const uint32_t row0 = tr.row0, rows = tr.rows;
  const uint32_t n0 = row0 / seq_rows, nseq = (row0 + rows - 1) / seq_rows - n0 + 1;
  const uint32_t prefix_limit = __builtin_amdgcn_readfirstlane(prefix_keys(a, g));
  // Where a part's keys and values are: the prompt, or one sequence's own.
  struct Source {
    const char *k, *v;
    uint32_t k_step, v_step;  // bytes from slot to slot
    const uint8_t *k_power, *v_power;
    uint32_t k_power_step, v_power_step;
  };
  constexpr int SIZE = BYTES ? 1 : sizeof(Elem);
  Source source{};  // of the tile that was asked for last
  auto set_source = [&](const KeyValues& kv, int64_t n) {
    Source& x = source;
    x.k = (const char*)kv.k + SIZE * ((int64_t)g * kv.k_s[0] + n * kv.k_s[1] + (int64_t)hk * kv.k_s[2]);
    x.v = (const char*)kv.v + SIZE * ((int64_t)g * kv.v_s[0] + n * kv.v_s[1] + (int64_t)hk * kv.v_s[2]);
    x.k_step = (uint32_t)(SIZE * kv.k_s[3]);
    x.v_step = (uint32_t)(SIZE * kv.v_s[3]);
    if (BYTES) {
      x.k_power = kv.k_scale + ((int64_t)g * kv.k_scale_s[0] + n * kv.k_scale_s[1] + (int64_t)hk * kv.k_scale_s[2]);
      x.v_power = kv.v_scale + ((int64_t)g * kv.v_scale_s[0] + n * kv.v_scale_s[1] + (int64_t)hk * kv.v_scale_s[2]);
      x.k_power_step = (uint32_t)kv.k_scale_s[3];
      x.v_power_step = (uint32_t)kv.v_scale_s[3];
    }
  };
  // Tiles of keys, in turn: `step` apart.
  const uint32_t first = BY_KEYS ? split * S::WAVES + wave : split, step = BY_KEYS ? splits * S::WAVES : splits;
  struct Part {
    uint32_t k0, limit, n;  // the tile's first key, its part's end, and the sequence (2^32 - 1: the prompt)
  };
  const uint32_t prefix_tiles = (prefix_limit + KT - 1) / KT;
  set_source(a.prefix, 0);

  char(*slab)[2][S::TILE] = lds[BY_KEYS ? wave : 0];
  const uint32_t loader = BY_KEYS ? 0 : wave;
  // A tile's loads, keys before values, 64 chunks each.
  constexpr int OF_KEYS = KT * CH, LOADS = 2 * OF_KEYS / 64 / S::LOADERS;  // OF_KEYS: chunks
  static_assert(2 * OF_KEYS % (64 * S::LOADERS) == 0 && (STORE == kCodes || OF_KEYS % 64 == 0), "loads");
  // Row and chunk of a lane's i-th load. Keys past the part's end are the last one again: their weights are 0, and what these
  // multiply is finite where the last key's values are. Chunks past the width are the row's first: finite where the row is,
  // and multiplied by 0 (keys) or not stored (values).
  constexpr int PER_CHUNK = STORE == kCodes ? 16 : 16 / sizeof(Elem);
  auto place = [&](int i, uint32_t last, uint32_t& r, uint32_t& c) {
    const uint32_t slot = ((i * S::LOADERS + loader) * 64 + lane) % OF_KEYS, row = slot / CH;
    c = (slot % CH) ^ (STORE == kCodes ? swizzle_codes<CH>(row) : swizzle<CH>(row));
    if (c * PER_CHUNK >= (uint32_t)a.width) c = 0;
    r = row < last ? row : last;
  };
  // A wave's first half of loads is of keys, the others of values, where that comes out even.
  constexpr bool EVEN = OF_KEYS % (64 * S::LOADERS) == 0;
  auto of_values = [&](int i) { return EVEN ? i >= LOADS / 2 : (i * S::LOADERS + loader) * 64 + lane >= OF_KEYS; };
  auto load_direct = [&](const Part& p, int stage) {
    const uint32_t k_step = source.k_step, v_step = source.v_step;
    const char* const k = source.k + (uint64_t)p.k0 * k_step;
    const char* const v = source.v + (uint64_t)p.k0 * v_step;
    const uint32_t to0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&slab[stage][0][0]);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t to = to0 + (i * S::LOADERS + loader) * 1024;
      uint32_t r, c;
      place(i, p.limit - 1 - p.k0, r, c);
      if (EVEN) {
        to_lds<false>(of_values(i) ? v : k, r * (of_values(i) ? v_step : k_step) + c * 16, to);
      } else {
        to_lds((of_values(i) ? v : k) + (uint64_t)r * (of_values(i) ? v_step : k_step) + c * 16, to);
      }
    }
  };
  // Powers of two of a tile's codes, key lane % 32.
  struct Powers {
    uint32_t k, v;
  };
  auto load_powers = [&](const Part& p) {
    Powers x{};
    if constexpr (STORE == kCodes) {
      const uint32_t last = p.limit - 1 - p.k0, r = p.k0 + ((lane & 31) < last ? (lane & 31) : last);
      x.k = source.k_power[(uint64_t)r * source.k_power_step];
      x.v = source.v_power[(uint64_t)r * source.v_power_step];
    }
    return x;
  };
  // 8-bit codes go through registers, where each becomes an element times its row's power of two (exactly).
  using Code = std::conditional_t<sizeof(Elem) == 2, u32x2, uint32_t>;
  struct Staged {
    Code code[STORE == kConverted ? LOADS : 1];
    uint32_t power[STORE == kConverted ? LOADS : 1];
  };
  auto load_codes = [&](const Part& p, Staged& s) {
    const char *const k = source.k, *const v = source.v;
    const uint8_t *const k_power = source.k_power, *const v_power = source.v_power;
    const uint32_t k_step = source.k_step, v_step = source.v_step, k_power_step = source.k_power_step, v_power_step = source.v_power_step;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint32_t r, c;
      place(i, p.limit - 1 - p.k0, r, c);
      const uint64_t key = p.k0 + r;
      s.code[i] = *(const Code*)((of_values(i) ? v : k) + key * (of_values(i) ? v_step : k_step) + c * PER_CHUNK);
      s.power[i] = (of_values(i) ? v_power : k_power)[key * (of_values(i) ? v_power_step : k_power_step)];
    }
  };
  auto put_codes = [&](const Staged& s, int stage) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *(u32x4*)(&slab[stage][0][0] + ((i * S::LOADERS + loader) * 64 + lane) * 16) = Op<T>::widen(s.code[i], __uint_as_float(s.power[i] << 23));
  };

  // A first tile of the prompt can be sent for before anything else is known.
  Part now{first * KT, prefix_limit, ~0u};
  const bool early = first < prefix_tiles;
  if constexpr (STORE != kConverted)
    if (early) load_direct(now, 0);

  // This lane's query.
  const uint32_t lane_row = (BY_KEYS ? 0 : wave * 32) + (lane & 31);
  const bool live = lane_row < rows;
  const uint32_t row = row0 + (live ? lane_row : 0), n_row = row / seq_rows, t_row = row % seq_rows / shared, h_row = hk * shared + row % shared;
  const int64_t q_at = (int64_t)g * a.q_s[0] + (int64_t)n_row * a.q_s[1] + (int64_t)h_row * a.q_s[2] + (int64_t)t_row * a.q_s[3];
  Frag qf[S::STEPS];
#pragma unroll
  for (int s = 0; s < S::STEPS; ++s) {
    // codes are read 16 at a time, for two steps
    const uint32_t col = STORE == kCodes ? 16 * (2 * (s / 2) + half) + 8 * (s % 2) : 16 * s + 8 * half;
    qf[s] = Frag(Elem(0.f));
    if (live && col < (uint32_t)a.width) qf[s] = *(const Frag*)((const Elem*)a.q + q_at + col);
  }

  const uint32_t own_limit = live ? own_keys(a, g, n_row, t_row) : 0;
  // Lane i: what is looked at of the tile's i-th sequence, and how many tiles of keys there are up to its end.
  const uint32_t n1 = n0 + nseq - 1;
  uint32_t limit_here = 0;
  if (lane < nseq) limit_here = own_keys(a, g, n0 + lane, n0 + lane == n1 ? (row0 + rows - 1) % seq_rows / shared : a.length - 1);
  uint32_t end_here = (limit_here + KT - 1) / KT + (lane == 0 ? prefix_tiles : 0);
  for (uint32_t d = 1; d < nseq; d *= 2) {
    const uint32_t x = __shfl_up(end_here, d);
    if (lane >= d) end_here += x;
  }
  const uint32_t key_tiles = __builtin_amdgcn_readlane(end_here, nseq - 1);
  uint32_t at_seq = 0, part_begin = 0, part_end = prefix_tiles, part_limit = prefix_limit;
  auto part_of = [&](uint32_t i) {
    if (i >= part_end) {
      do {
        part_begin = part_end;
        part_end = __builtin_amdgcn_readlane(end_here, at_seq++);
      } while (i >= part_end);
      part_limit = __builtin_amdgcn_readlane(limit_here, at_seq - 1);
      set_source(a.own, n0 + at_seq - 1);
    }
    return Part{(i - part_begin) * KT, part_limit, at_seq ? n0 + at_seq - 1 : ~0u};
  };

  f32x16 o[S::PV];
#pragma unroll
  for (int d = 0; d < S::PV; ++d) o[d] = f32x16(0.f);
  float m = -INFINITY, l = 0.f;  // l: of this lane's keys
  const float c = a.scale * kLog2e;

  auto products = [&](const Part& p, int stage, const Powers& pow) {
    const uint32_t limit = p.n == ~0u ? prefix_limit : p.n == n_row ? own_limit : 0;
    if (__all(limit <= p.k0)) return;  // none of the wave's rows
    const char* kt = slab[stage][0];
    const char* vt = slab[stage][1];
    f32x16 s[NK];
    if constexpr (STORE == kCodes) {
      if (half == 0) powers[wave][lane] = power_of(pow.v);
      const float power = __uint_as_float((uint32_t)pow.k << 23);
      const uint32_t r = lane & 31;
      s[0] = f32x16(0.f);
#pragma unroll
      for (int q = 0; q < S::STEPS / 2; ++q) {
        uint32_t c = 2 * q + half;
        if (CH % 2) c = c < CH ? c : CH - 1;  // (multiplied by 0)
        const u32x4 codes = *(const u32x4*)(kt + r * CH * 16 + (c ^ swizzle_codes<CH>(r)) * 16);
        s[0] = Op<T>::mma(Op<T>::widen8(u32x2{codes[0], codes[1]}, power), qf[2 * q], s[0]);
        s[0] = Op<T>::mma(Op<T>::widen8(u32x2{codes[2], codes[3]}, power), qf[2 * q + 1], s[0]);
      }
    } else {
      // All of the tile's keys on their way, then products of two sums in turn: each waits for the one before it.
      constexpr int SUMS = NK == 1 ? 2 : NK;
      f32x16 sum[SUMS];
#pragma unroll
      for (int i = 0; i < SUMS; ++i) sum[i] = f32x16(0.f);
      Frag kf[S::STEPS][NK];
#pragma unroll
      for (int q = 0; q < S::STEPS; ++q)
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const uint32_t r = i * 32 + (lane & 31);
          if constexpr (!S::kWide) {
            kf[q][i] = *(const Frag*)(kt + r * CH * 16 + ((2 * q + half) ^ swizzle<CH>(r)) * 16);
          } else {
            const f32x4 lo = *(const f32x4*)(kt + r * CH * 16 + ((4 * q + 2 * half) ^ swizzle<CH>(r)) * 16);
            const f32x4 hi = *(const f32x4*)(kt + r * CH * 16 + ((4 * q + 2 * half + 1) ^ swizzle<CH>(r)) * 16);
            kf[q][i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          }
        }
      if (!S::kWide) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < S::STEPS; ++q)
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          f32x16& to = sum[NK == 1 ? q % 2 : i];
          to = Op<T>::mma(kf[q][i], qf[q], to);
        }
#pragma unroll
      for (int i = 0; i < NK; ++i) s[i] = NK == 1 ? sum[0] + sum[1] : sum[i];
    }
    // Values of 16 keys, for all columns.
    constexpr int GROUPS = 2 * NK;
    using Read = std::conditional_t<STORE == kCodes, u32x2, FragV>;
    Read values[2][S::PV];
    auto read_group = [&](int g) {
#pragma unroll
      for (int d = 0; d < S::PV; ++d) {
        Read& to = values[g % 2][d];
        if constexpr (STORE == kCodes) {
          // eight rows of 16 codes for each 16 lanes, which get a column each
          const uint32_t of = 2 * d + (lane & 31) / 16, chunk = of < CH ? of : CH - 1, j = (lane & 15) / 2;
          const uint32_t r = g * 16 + j / 4 * 8 + 4 * half + j % 4;
          typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
          to = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) i32x2*)(vt + r * CH * 16 + (chunk ^ swizzle_codes<CH>(r)) * 16 + (lane & 1) * 8)));
        } else if constexpr (!S::kWide) {
          // four rows of 16 columns for each 16 lanes, which get a column each
          const uint32_t col = 32 * d + (lane & 31) / 16 * 16, group = col / 8 < CH ? col / 8 : CH - 2, chunk = group + (lane & 3) / 2;
          s16x4 part[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t r = g * 16 + j * 8 + 4 * half + (lane & 15) / 4;
            part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + r * CH * 16 + (chunk ^ swizzle<CH>(r)) * 16 + (lane & 1) * 8));
          }
          to = __builtin_bit_cast(FragV, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
          const uint32_t col = 32 * d + (lane & 31), chunk = col / 4 < CH ? col / 4 : CH - 1;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t r = g * 16 + j / 4 * 8 + 4 * half + j % 4;
            to[j] = *(const float*)(vt + r * CH * 16 + (chunk ^ swizzle<CH>(r)) * 16 + (lane & 3) * 4);
          }
        }
      }
    };
    read_group(0);
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
    if (__any(top > m + kLag)) {
      const float m2 = fmaxf(m, top);
      const float f = m2 == -INFINITY ? 1.f : exp2_hw(m - m2);
      m = m2;
      l *= f;
#pragma unroll
      for (int d = 0; d < S::PV; ++d) o[d] *= f;
    }
    const float mm = m == -INFINITY ? 0.f : m - kBias;
    // Weights of 16 keys at a time (those of 8 a lane), each next to the products with the 16 before: their values are read one such
    // group ahead.
    FragV w[GROUPS], rest[kTwo ? GROUPS : 1];
    auto weights = [&](int g) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int of = g % 2 * 2 + b;
        f32x4 power;
        if (STORE == kCodes) power = *(const f32x4*)&powers[wave][8 * of + 4 * half];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float e = exp2_hw(__builtin_fmaf(s[g / 2][4 * of + r], c, -mm));
          l += e;
          if (STORE == kCodes) e *= power[r];
          w[g][4 * b + r] = (typename TV::Elem)e;
          if constexpr (kTwo) rest[g][4 * b + r] = (typename TV::Elem)(e - (float)w[g][4 * b + r]);
        }
      }
    };
    weights(0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + 1 < GROUPS) read_group(g + 1);
#pragma unroll
      for (int d = 0; d < S::PV; ++d) {
        if constexpr (STORE == kCodes) {
          const FragV v = Op<TV>::widen8(values[g % 2][d], 1.f);
          o[d] = Op<TV>::mma(v, w[g], o[d]);
          if constexpr (kTwo) o[d] = Op<TV>::mma(v, rest[g], o[d]);
        } else o[d] = Op<TV>::mma(values[g % 2][d], w[g], o[d]);
      }
      if (g + 1 < GROUPS) weights(g + 1);
      if (!S::kWide) __builtin_amdgcn_sched_barrier(0);
    }
  };

  // No load or read of LDS is left open, and (tiles of several waves) every wave is here.
  auto arrive_all = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
    if (!BY_KEYS) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (first < key_tiles) {
    if (!early || STORE == kConverted) now = part_of(first);
    Staged st;
    Powers pow = load_powers(now);
    if constexpr (STORE == kConverted) {
      load_codes(now, st);
      put_codes(st, 0);
    } else if (!early) {
      load_direct(now, 0);
    }
    int stage = 0;
    for (uint32_t i = first; i < key_tiles; i += step) {
      const bool more = i + step < key_tiles;
      Part next = now;
      Powers next_pow = pow;
      if (more) next = part_of(i + step);
      arrive_all();
      if (more) {
        // where there is room the next tile is on its way while this one's products run
        next_pow = load_powers(next);
        if constexpr (STORE == kConverted) load_codes(next, st);
        else if (S::STAGES == 2) load_direct(next, stage ^ 1);
      }
      products(now, stage, pow);
      if constexpr (S::STAGES == 1) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);  // what was read of the tile is here
        asm volatile("" ::: "memory");
      }
      if (more) {
        if constexpr (STORE == kConverted) put_codes(st, S::STAGES == 1 ? 0 : stage ^ 1);
        else if (S::STAGES == 1) load_direct(next, 0);
      }
      if (S::STAGES == 2) stage ^= 1;
      now = next;
      pow = next_pow;
    }
  }
  l = both_halves(l, [](float x, float y) { return x + y; });
  m -= kBias;  // what the sums are relative to

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
    static_assert((S::WAVES - 1) * 32 * PITCH * 4 <= (int)sizeof(lds), "room");
    float* mine = (float*)lds + (wave - 1) * 32 * PITCH;
#pragma unroll
    for (int d = 0; d < S::PV; ++d) o[d] *= f;
    if (wave > 0)
#pragma unroll
      for (int d = 0; d < S::PV; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *(f32x4*)(mine + (lane & 31) * PITCH + 32 * d + 8 * b + 4 * half) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    __syncthreads();
    if (wave != 0) return;  // (the sums that are left take one wave)
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f32x4 x = f32x4(0.f);
#pragma unroll
        for (int i = 0; i < S::WAVES - 1; ++i) x += *(const f32x4*)((float*)lds + (i * 32 + (lane & 31)) * PITCH + 32 * d + 8 * b + 4 * half);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][4 * b + r] += x[r];
      }
  }
  float zero = 0.f;  // NaN where a sum is not finite (columns past the width are, or are the row's first ones again)
#pragma unroll
  for (int d = 0; d < S::PV; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) zero = __builtin_fmaf(o[d][j], 0.f, zero);
  const bool finite = zero == 0.f;
  const uint64_t lone_lanes = __ballot(live && !finite);
  const uint32_t lone = (uint32_t)lone_lanes | (uint32_t)(lone_lanes >> 32);
  if (lone) lone_rows<T, BY_KEYS, BYTES, KT, S::WAVES>(BY_KEYS ? 0 : wave * 32, lone);
  if (!live || lone >> (lane & 31) & 1) return;
  if (splits > 1) {
    const uint64_t to_row = partial_row(plan, item, lane_row);
    if (half == 0) call.partial_ms[to_row] = float2{m, l};
    float* to = call.partial + to_row * a.width;
#pragma unroll
    for (int d = 0; d < S::PV; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t col = 32 * d + 8 * b + 4 * half;
        if (col < (uint32_t)a.width) *(f32x4*)(to + col) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
      }
    return;
  }
  // (a query all of whose keys score -inf has no answer: 0 / 0)
  const float inv = prefix_limit + own_limit == 0 ? 0.f : 1.f / l;
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

// The splits' sums of each row of a tile, joined. 32 lanes a row, four columns a lane.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(Attend a, AttendPlan plan, const float* partial, const float2* partial_ms) {
  using Elem = typename T::Elem;
  const uint32_t shared = a.heads / a.kv_heads, seq_rows = (uint32_t)a.length * shared, all_rows = seq_rows * a.sequences;
  const uint32_t each = (plan.tile_rows + 7) / 8, index = blockIdx.x / each, lane_row = blockIdx.x % each * 8 + threadIdx.x / 32;
  const uint32_t item = index / plan.tail * plan.per + plan.whole + index % plan.tail, col = threadIdx.x % 32 * 4;
  if (item >= (uint32_t)plan.items) return;
  const TileRows t = tile_rows_of(plan, plan.tiles - 1 - item % plan.tiles, seq_rows, all_rows);
  if (lane_row >= t.rows || col >= (uint32_t)a.width) return;
  const uint64_t from = (uint64_t)index * plan.splits * plan.tile_rows + lane_row;
  float m = -INFINITY;
  for (int i = 0; i < plan.splits; ++i) m = fmaxf(m, partial_ms[from + (uint64_t)i * plan.tile_rows].x);
  float l = 0.f;
  f32x4 o = f32x4(0.f);
  auto add = [&](int i) {
    const uint64_t at = from + (uint64_t)i * plan.tile_rows;
    const float2 ms = partial_ms[at];
    const f32x4 x = *(const f32x4*)(partial + at * a.width + col);
    const float f = ms.x == -INFINITY ? 0.f : exp2_hw(ms.x - m);  // (saw no key)
    l = __builtin_fmaf(ms.y, f, l);
    o += x * f;
  };
#pragma unroll 4
  for (int i = 0; i < plan.splits; ++i) add(i);
  const f32x4 nothing = o - o;
  if (nothing[0] + nothing[1] + nothing[2] + nothing[3] != 0.f) {  // not finite: the sums of up to 64 finite parts are, as 2^-8 of themselves
    m += 8.f;
    l = 0.f;
    o = f32x4(0.f);
#pragma unroll 1
    for (int i = 0; i < plan.splits; ++i) add(i);
  }
  const uint32_t gh = item / plan.tiles, row = t.row0 + lane_row, g = gh / a.kv_heads, h = gh % a.kv_heads * shared + row % shared;
  const float inv = prefix_keys(a, g) + own_keys(a, g, row / seq_rows, row % seq_rows / shared) == 0 ? 0.f : 1.f / l;
  typedef Elem Quad __attribute__((ext_vector_type(4)));
  *(Quad*)((Elem*)a.out + (int64_t)g * a.out_s[0] + (int64_t)(row / seq_rows) * a.out_s[1] + (int64_t)h * a.out_s[2] +
           (int64_t)(row % seq_rows / shared) * a.out_s[3] + col) = Quad{(Elem)(o[0] * inv), (Elem)(o[1] * inv), (Elem)(o[2] * inv), (Elem)(o[3] * inv)};
}

template <class T, int QS, bool BY_KEYS, Store STORE, int WAVES>
void launch_one(const Attend& a, const AttendPlan& p, float* partial, float2* ms, hipStream_t st) {
  attend_kernel<T, QS, BY_KEYS, STORE, WAVES><<<8 * (p.whole + p.tail * p.splits), 64 * WAVES, 0, st>>>(Call{a, p, partial, ms});
}
template <class T, int QS, Store STORE>
void launch_by_keys(const Attend& a, const AttendPlan& p, float* partial, float2* ms, hipStream_t st) {
  if (p.waves == 1) launch_one<T, QS, true, STORE, 1>(a, p, partial, ms, st);
  else if (p.waves == 2) launch_one<T, QS, true, STORE, 2>(a, p, partial, ms, st);
  else launch_one<T, QS, true, STORE, 4>(a, p, partial, ms, st);
}
template <class T, int QS>
void launch_qs(const Attend& a, const AttendPlan& p, float* partial, float2* ms, hipStream_t st) {
  if (p.by_keys) {
    if (!a.bytes) launch_by_keys<T, QS, kOperands>(a, p, partial, ms, st);
    else if (a.whole_chunks) launch_by_keys<T, QS, kCodes>(a, p, partial, ms, st);
    else launch_by_keys<T, QS, kConverted>(a, p, partial, ms, st);
  } else {
    if (!a.bytes) launch_one<T, QS, false, kOperands, 4>(a, p, partial, ms, st);
    else launch_one<T, QS, false, kConverted, 4>(a, p, partial, ms, st);
  }
}
template <class T>
hipError_t launch_typed(const Attend& a, const AttendPlan& p, void* workspace, hipStream_t st) {
  const uint64_t rows = 8ull * p.tail * p.splits * p.tile_rows;
  float2* ms = (float2*)workspace;
  float* partial = (float*)((char*)workspace + (rows * 8 + 15) / 16 * 16);
  const int qs = (a.width + 15) / 16;
  if (qs <= 4) launch_qs<T, 4>(a, p, partial, ms, st);
  else if (qs == 5) launch_qs<T, 5>(a, p, partial, ms, st);
  else if (qs == 6) launch_qs<T, 6>(a, p, partial, ms, st);
  else launch_qs<T, 8>(a, p, partial, ms, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.tail == 0) return e;
  join_kernel<T><<<8 * p.tail * ((p.tile_rows + 7) / 8), 256, 0, st>>>(a, p, partial, ms);
  return hipGetLastError();
}

}  // namespace

AttendPlan attend_plan(int dtype, const Attend& a) {
  const int64_t shared = a.heads / a.kv_heads, seq_rows = a.length * shared, heads = (int64_t)a.groups * a.kv_heads;
  AttendPlan p{};
  // Waves that take keys for themselves, 32 rows a workgroup, or tiles of 128 rows that share keys. The first reads keys four times as often for
  // the same rows, and leaves fewer rows empty and more workgroups to run. Sequences of
  //   up to 16 rows: the first (32 x 16 rows after 1,000 keys, fp16 heads of 128: 81 us, shared 85);
  //   up to 96 rows, in no more than one round of workgroups, or after few keys: the first (34 heads of 40 rows after 5,066 keys: fp32 92 us,
  //   shared 164; 32 x 40 rows after 122, bf16: 29 and 29, after 600: 71 and 56; fp32 after 600: 309 and 412);
  //   more: the second (one sequence of 128 rows after 5,066: 37 and 35; fp32 211 and 169).
  // Codes are converted by each wave for itself in the first, without a stop in registers before: of wide heads it is the faster one
  // throughout (a causal 2,048 of 40 heads of 128: 95 us in bf16 and 109 in fp16, shared 164; heads of 80, 16 x 256: 33 and 31).
  const int64_t keys_of_one = a.prefix_slots + a.slots, own_tiles = heads * a.sequences * ((seq_rows + 31) / 32);
  const int64_t few_keys = seq_rows <= 32 || dtype == 0 || a.bytes ? 1000 : 256;
  p.by_keys = seq_rows <= 16 || (a.bytes && a.width >= 96 && a.width % 16 == 0) || (seq_rows <= 96 && (own_tiles <= 512 || keys_of_one < few_keys));
  const int64_t most = p.by_keys ? 32 : 128;
  if (seq_rows <= most) {
    p.tile_rows = (int32_t)(most / seq_rows * seq_rows);
    if (p.tile_rows > seq_rows * a.sequences) p.tile_rows = (int32_t)(seq_rows * a.sequences);
    p.tiles = (int32_t)((seq_rows * a.sequences + p.tile_rows - 1) / p.tile_rows);
  } else {
    p.tile_rows = (int32_t)most;
    p.tiles = (int32_t)((seq_rows + most - 1) / most * a.sequences);
  }
  const int64_t items = heads * p.tiles;
  if (items > (int64_t)1 << 23) {  // (refused)
    p.items = INT32_MAX;
    return p;
  }
  p.items = (int32_t)items;
  p.per = (p.items + 7) / 8;
  // An XCD's 32 compute units run `slots` workgroups at a time. Items beyond a multiple of that would leave most of them idle for as long as
  // one takes: as many parts of them as fill the slots once (40 heads of 128, fp16, keys that the caches hold: 64 single tokens after
  // 2,048 keys 26 us, whole items 38; 128 tokens after 8,192: 47 and 164). A part has 256 keys or more (one token after 500: 12.6 us in two
  // parts, 11.6 whole). Shared tiles of 16-bit operands keep a compute unit's matrix units busy by one workgroup, and a part's sums are 128
  // rows that are written and read again: one a compute unit (128 tokens after 8,192: 47 us, two 50; a causal 1,000 of 40 heads of 128: 39
  // and 40; 8 x 60 tokens after 1,000: 30 and 35). fp32 and codes
  // that are converted on the way take two (16 x 60 tokens after 3,000, fp32: 106 us, one 131; 32 x 61 after 2,048 from
  // codes 225 and 243).
  const int64_t seqs = p.tile_rows > seq_rows ? p.tile_rows / seq_rows : 1, keys = a.prefix_slots + seqs * a.slots;
  // Of the 256 waves that an XCD holds (wide fp32 heads: 128), an item of few keys takes as many as let all items run at once: a second round
  // begins again with lengths and first keys (32 x 6 rows after 122 keys, 640 items: two waves 13.8 us, four 20.6, one 15.4; 64 x 12
  // causal, 2,048 items: one wave 9.6, four 28.7). Many keys are worth four (512 single tokens after 2,000: 374 us, two 392).
  const int held = p.by_keys && dtype == 0 && a.width > 64 ? 128 : 256;
  p.waves = 4;
  if (p.by_keys && keys < 1024)
    while (p.waves > 1 && p.per * p.waves > held) p.waves /= 2;
  const int slots = p.by_keys ? held / p.waves : dtype != 0 && !a.bytes ? 32 : 64;
  const int rest = p.per % slots;
  const int64_t fit = rest ? slots / rest : 1, cap = keys / 256;
  p.splits = (int32_t)(fit < cap ? fit : cap);
  if (p.splits < 2) p.splits = 1;
  p.tail = p.splits > 1 ? rest : 0;
  p.whole = p.per - p.tail;
  return p;
}

int64_t attend_workspace(const Attend& a, const AttendPlan& p) {
  const int64_t rows = (int64_t)8 * p.tail * p.splits * p.tile_rows;
  return (rows * 8 + 15) / 16 * 16 + rows * a.width * 4;
}

hipError_t launch_attend(int dtype, const Attend& a, const AttendPlan& p, void* workspace, hipStream_t st) {
  switch (dtype) {
    case 0: return launch_typed<TypeF32>(a, p, workspace, st);
    case 1: return launch_typed<TypeF16>(a, p, workspace, st);
    default: return launch_typed<TypeBF16>(a, p, workspace, st);
  }
}

}  // namespace dz
