// What the kernels of attention over a shared prompt have in common.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "dz_prefix.h"
#include "dz_token_math.h"

namespace dz {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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
  __device__ static Frag widen8(u32x2 c, float scale) { return __builtin_bit_cast(Frag, widen(c, scale)); }
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
  __device__ static Frag widen8(u32x2 c, float scale) { return __builtin_bit_cast(Frag, widen(c, scale)); }
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
  __device__ static Frag widen8(u32x2 c, float scale) {
    return __builtin_shufflevector(__builtin_bit_cast(f32x4, widen(c[0], scale)), __builtin_bit_cast(f32x4, widen(c[1], scale)), 0, 1, 2, 3, 4, 5, 6, 7);
  }
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
// at one chunk (a read of keys), and the rows and chunks of 32 lanes' read of values, then lie in different banks, or in few of
// the same.
template <int CH>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  if (CH == 8) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
  if (CH == 10) return r >> 3 & 1;
  if (CH == 12 || CH == 20) return r >> 2 & 3;
  if (CH == 24) return r >> 1 & 7;
  return (r & 3) << 2 | (r >> 2 & 3);
}
// The same of rows of CH chunks of 16 codes.
template <int CH>
__device__ __forceinline__ uint32_t swizzle_codes(uint32_t r) {
  if (CH == 4) return r >> 2 & 3;
  if (CH == 5) return 0;
  if (CH == 6) return r >> 3 & 1;
  return (r >> 1 & 1) << 1 | (r >> 3 & 1) << 2 | (r >> 2 & 1);
}

// The rows of a tile: whole sequences, or rows of one.
struct TileRows {
  uint32_t row0, rows;
};
__device__ __forceinline__ TileRows tile_rows_of(const AttendPlan& plan, uint32_t tile, uint32_t seq_rows, uint32_t all_rows) {
  const uint32_t most = plan.tile_rows;
  if (most >= seq_rows) {
    const uint32_t row0 = tile * most;
    return {row0, all_rows - row0 < most ? all_rows - row0 : most};
  }
  const uint32_t per_seq = (seq_rows + most - 1) / most, r = tile % per_seq * most;
  return {tile / per_seq * seq_rows + r, seq_rows - r < most ? seq_rows - r : most};
}

// What a workgroup takes of a call.
struct Item {
  uint32_t xcd, at;         // its XCD, and its place among that one's items
  uint32_t split, splits;   // its part of the keys
  uint32_t gh, g, hk, tile;  // group and key head, and the tile of their rows
};
// Workgroups go to the 8 XCDs in turn: each XCD takes consecutive items, whose keys its L2 holds for them.
__device__ __forceinline__ bool item_of(const Attend& a, const AttendPlan& plan, Item& x) {
  const uint32_t order = blockIdx.x / 8, after = order - plan.whole;
  const bool parted = order >= (uint32_t)plan.whole;
  x.xcd = blockIdx.x % 8;
  x.at = parted ? plan.whole + after / plan.splits : order;
  const uint32_t item = x.xcd * plan.per + x.at;
  x.split = parted ? after % plan.splits : 0;
  x.splits = parted ? plan.splits : 1;
  x.gh = item / plan.tiles;
  x.tile = plan.tiles - 1 - item % plan.tiles;  // the longest first
  x.g = x.gh / a.kv_heads;
  x.hk = x.gh % a.kv_heads;
  return x.at < (uint32_t)plan.per && item < (uint32_t)plan.items;
}
// Where the sums of a tile's row go until they are joined.
__device__ __forceinline__ uint64_t partial_row(const AttendPlan& plan, const Item& x, uint32_t row) {
  return (((uint64_t)x.xcd * plan.tail + x.at - plan.whole) * x.splits + x.split) * plan.tile_rows + row;
}

}  // namespace dz
