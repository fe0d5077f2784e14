// Internal interface between the C ABI of attention over a shared prompt and of
// the 8-bit cache (dz_prefix_api.hip) and their kernels (dz_attention.hip,
// dz_cache.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dz {

// Keys and values by strides in elements (bytes of an 8-bit store): group,
// sequence, head, slot. The width is contiguous. Scales (8-bit stores) are
// e8m0, one byte for each slot of a head.
struct KeyValues {
  const void* k;
  const void* v;
  int64_t k_s[4], v_s[4];
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  int64_t k_scale_s[4], v_scale_s[4];
};

struct Attend {
  const void* q;
  void* out;
  int64_t q_s[4], out_s[4];  // group, sequence, head, token
  KeyValues own, prefix;     // prefix: its sequence stride is not used
  const int32_t* positions;       // (groups, sequences); NULL: slots - length
  const int32_t* prefix_lengths;  // (groups); NULL: prefix_slots
  int32_t groups, sequences, heads, kv_heads, length, width, slots, prefix_slots;
  int32_t bytes;  // an 8-bit store
  int32_t whole_chunks;  // whose rows are whole chunks of 16 codes, at multiples of 16 bytes
  float scale;
};

// How a call is cut. An item is a tile of up to tile_rows rows of one key head. Each of the 8 XCDs takes `per` items one
// after another: first `whole` of them, a workgroup each, then `tail`, of which `splits` workgroups each take a part of the keys.
struct AttendPlan {
  bool by_keys;  // a workgroup's waves share its rows and take keys in turn; else they share keys
  int32_t waves;  // of a workgroup
  int32_t tile_rows, tiles;
  int32_t items, per, whole, tail, splits;
};
AttendPlan attend_plan(int dtype, const Attend& a);
int64_t attend_workspace(const Attend& a, const AttendPlan& p);
hipError_t launch_attend(int dtype, const Attend& a, const AttendPlan& p, void* workspace, hipStream_t st);

struct CacheRows {
  const void* x[2];  // keys and values: (batch, head, token, width), the width contiguous
  int64_t x_s[2][3];
  void* code[2];
  int64_t code_s[2][3];
  void* scale[2];
  int64_t scale_s[2][3];
  const int32_t* positions;  // (batch); NULL: `position`
  int32_t position;
  int32_t batch, heads, length, width, slots;
};
// x is read and the cache written, or (read) the other way round.
hipError_t launch_cache(int dtype, const CacheRows& a, bool read, hipStream_t st);

}  // namespace dz
