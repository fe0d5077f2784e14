// An 8-bit store of keys and values: e4m3 codes with one power of two for each
// token and head.
//
// x is kept as code 2^e, with e the least that leaves no value of the row above 448, e4m3's largest, and code the
// nearest e4m3 number to x / 2^e (ties to even). A power of two moves nothing but exponents: x / 2^e and code 2^e are
// exact, so the only rounding is the code's, of half a unit of 3 bits (2^-4 of the value; 2^-10 2^e below 2^-6 2^e), and an
// arbitrary scale would save none of it.
//
// Bound by memory: 2,048 tokens of 40 heads of 128 written in 15 us (63 MB; 12.7 at a large copy's 4.96 TB/s), 64 x 300 read in
// 82 us (591 MB, 7.2 TB/s with what the caches hold); one token of 64 sequences 3.5 us, a launch.
#include "dz_prefix.h"
#include "dz_token_math.h"

namespace dz {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The least power kept: rows of smaller numbers lose bits, or become 0 (largest value under 2^-101).
constexpr int kLeastPower = -100;
// The largest value kept: one above 240 2^8 could round to 2^16, which fp16 does not have, and one above 240 2^120 to 2^128, which neither
// of the others has.
template <class T>
constexpr float kLargest = __is_same(T, TypeF16) ? 61440.f : 0x1.ep127f;

constexpr int kThreads = 256;

// LANES lanes a row, 8 elements each; a thread takes EACH rows, whose loads are all on their way before the first is used.
// Keys in the grid's first plane, values in its second. Rows go along the store, a head's slots next to each other: its
// lines and scales are whole then, and the other side's rows are 16 to 512 consecutive bytes in either order.
template <class T, bool READ, int LANES, int EACH>
__global__ __launch_bounds__(kThreads) void cache_kernel(CacheRows a) {
  using Elem = typename T::Elem;
  typedef Elem Eight __attribute__((ext_vector_type(8)));
  constexpr uint32_t ROWS = kThreads / LANES;
  const uint32_t rows = (uint32_t)a.batch * a.length * a.heads, which = blockIdx.y;
  const uint32_t col = threadIdx.x % LANES * 8;
  const int64_t* const xs = a.x_s[which];
  const int64_t* const cs = a.code_s[which];
  const int64_t* const ss = a.scale_s[which];
  const bool there = col < (uint32_t)a.width;
  bool live[EACH];
  Elem* x[EACH];
  uint8_t *code[EACH], *scale[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const uint32_t i = (blockIdx.x * EACH + r) * ROWS + threadIdx.x / LANES;
    const uint32_t bh = i / a.length, t = i - bh * a.length, b = bh / a.heads, h = bh - b * a.heads;
    live[r] = i < rows;
    int64_t slot = 0;
    if (live[r]) {
      slot = (int64_t)(a.positions ? a.positions[b] : a.position) + t;
      live[r] = slot >= 0 && slot < a.slots;
    }
    x[r] = (Elem*)a.x[which] + (int64_t)b * xs[0] + (int64_t)h * xs[1] + (int64_t)t * xs[2] + col;
    code[r] = (uint8_t*)a.code[which] + (int64_t)b * cs[0] + (int64_t)h * cs[1] + slot * cs[2] + col;
    scale[r] = (uint8_t*)a.scale[which] + (int64_t)b * ss[0] + (int64_t)h * ss[1] + slot * ss[2];
  }
  if constexpr (READ) {
    u32x2 c[EACH];
    uint8_t e[EACH];
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (live[r] && there) {
        c[r] = *(const u32x2*)code[r];
        e[r] = *scale[r];
      }
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (live[r] && there) {
        const float f = __uint_as_float((uint32_t)e[r] << 23);
        Eight v;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[r][j], f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[r][j], f, true);
          v[4 * j] = (Elem)lo[0];
          v[4 * j + 1] = (Elem)lo[1];
          v[4 * j + 2] = (Elem)hi[0];
          v[4 * j + 3] = (Elem)hi[1];
        }
        __builtin_nontemporal_store(v, (Eight*)x[r]);
      }
  } else {
    Eight in[EACH];
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      in[r] = Eight(Elem(0.f));
      if (live[r] && there) in[r] = *(const Eight*)x[r];
    }
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      float v[8];
      uint32_t most = 0;  // bits of the largest magnitude: NaN above infinity above numbers
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = (float)in[r][j];
        const uint32_t m = __float_as_uint(v[j]) & 0x7fffffffu;
        most = m > most ? m : most;
      }
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) {
        const uint32_t o = __shfl_xor(most, d);
        most = o > most ? o : most;
      }
      const bool finite = most < 0x7f800000u;
      if (__any(finite && most > __float_as_uint(kLargest<T>))) {  // (hardly any wave: a prompt's write in bf16 14.1 us, clamped throughout 14.9)
        if (finite && most > __float_as_uint(kLargest<T>)) most = __float_as_uint(kLargest<T>);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -kLargest<T>), kLargest<T>);
      }
      int e = (int)(most >> 23) - 135 + ((most & 0x7fffffu) > 0x600000u);
      e = most == 0 || !finite ? 0 : e < kLeastPower ? kLeastPower : e;
      const float f = __uint_as_float((uint32_t)(127 - e) << 23);
      u32x2 c;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = v[4 * j + k] * f;
        c[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
      }
      if (!finite) c = u32x2(0x7f7f7f7fu);
      if (live[r] && there) {
        *(u32x2*)code[r] = c;
        if (col == 0) *scale[r] = (uint8_t)(e + 127);
      }
    }
  }
}

template <class T, bool READ, int LANES>
void launch_lanes(const CacheRows& a, hipStream_t st) {
  const uint32_t rows = (uint32_t)a.batch * a.length * a.heads, each = kThreads / LANES;
  // four rows a thread where that leaves two workgroups a compute unit (64 x 300 tokens of 40 heads of 64 written: 59 us, one row a thread 76;
  // 64 tokens: one row a thread 3.0 us, four 4.5)
  if (rows >= 4 * each * 256) cache_kernel<T, READ, LANES, 4><<<dim3((rows + 4 * each - 1) / (4 * each), 2), kThreads, 0, st>>>(a);
  else cache_kernel<T, READ, LANES, 1><<<dim3((rows + each - 1) / each, 2), kThreads, 0, st>>>(a);
}
template <class T>
void launch_typed(const CacheRows& a, bool read, hipStream_t st) {
  if (a.width <= 64) read ? launch_lanes<T, true, 8>(a, st) : launch_lanes<T, false, 8>(a, st);
  else read ? launch_lanes<T, true, 16>(a, st) : launch_lanes<T, false, 16>(a, st);
}

}  // namespace

hipError_t launch_cache(int dtype, const CacheRows& a, bool read, hipStream_t st) {
  switch (dtype) {
    case 0: launch_typed<TypeF32>(a, read, st); break;
    case 1: launch_typed<TypeF16>(a, read, st); break;
    default: launch_typed<TypeBF16>(a, read, st);
  }
  return hipGetLastError();
}

}  // namespace dz
