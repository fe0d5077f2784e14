// An 8-bit store of keys and values: e4m3 codes with one power of two for each
// token and head.
//
// x is kept as code 2^e, with e the least that leaves no value of the row above 448, e4m3's largest, and code the
// nearest e4m3 number to x / 2^e (ties to even). A power of two moves nothing but exponents: x / 2^e and code 2^e are
// exact, so the only rounding is the code's, of half a unit of 3 bits (2^-4 of the value; 2^-10 2^e below 2^-6 2^e), and an
// arbitrary scale would save none of it.
#include "dz_prefix.h"
#include "dz_token_math.h"

namespace dz {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The least power kept: rows of smaller numbers lose bits, or become 0 (largest value under 2^-101).
constexpr int kLeastPower = -100;
// fp16 values above 61,440 would round to 65,536, which fp16 does not have.
constexpr float kLargestHalf = 61440.f;

constexpr int kRowLanes = 16;  // of 8 elements: a width of up to 128

template <class T, bool READ>
__global__ __launch_bounds__(256) void cache_kernel(CacheRows a) {
  using Elem = typename T::Elem;
  typedef Elem Eight __attribute__((ext_vector_type(8)));
  // Rows in the order of a projection's output, heads next to each other; keys, then values.
  const uint64_t rows = (uint64_t)a.batch * a.length * a.heads;
  const uint64_t at = (uint64_t)blockIdx.x * (256 / kRowLanes) + threadIdx.x / kRowLanes;
  const uint32_t col = threadIdx.x % kRowLanes * 8;
  if (at >= 2 * rows) return;
  const int which = at >= rows;
  const uint64_t i = at - which * rows;
  const uint32_t h = (uint32_t)(i % a.heads), t = (uint32_t)(i / a.heads % a.length), b = (uint32_t)(i / a.heads / a.length);
  const int64_t slot = (int64_t)(a.positions ? a.positions[b] : a.position) + t;
  if (slot < 0 || slot >= a.slots) return;
  const int64_t(&xs)[3] = a.x_s[which], (&cs)[3] = a.code_s[which], (&ss)[3] = a.scale_s[which];
  Elem* x = (Elem*)a.x[which] + (int64_t)b * xs[0] + (int64_t)h * xs[1] + (int64_t)t * xs[2] + col;
  uint8_t* code = (uint8_t*)a.code[which] + (int64_t)b * cs[0] + (int64_t)h * cs[1] + slot * cs[2] + col;
  uint8_t* scale = (uint8_t*)a.scale[which] + (int64_t)b * ss[0] + (int64_t)h * ss[1] + slot * ss[2];
  const bool there = col < (uint32_t)a.width;
  if constexpr (READ) {
    if (!there) return;
    const float f = __uint_as_float((uint32_t)*scale << 23);
    const u32x2 c = *(const u32x2*)code;
    Eight v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[j], f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[j], f, true);
      v[4 * j] = (Elem)lo[0];
      v[4 * j + 1] = (Elem)lo[1];
      v[4 * j + 2] = (Elem)hi[0];
      v[4 * j + 3] = (Elem)hi[1];
    }
    *(Eight*)x = v;
  } else {
    float v[8];
    uint32_t most = 0;  // bits of the largest magnitude: NaN above infinity above numbers
    if (there) {
      const Eight e = *(const Eight*)x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = (float)e[j];
        const uint32_t m = __float_as_uint(v[j]) & 0x7fffffffu;
        most = m > most ? m : most;
      }
    }
#pragma unroll
    for (int d = 1; d < kRowLanes; d *= 2) {
      const uint32_t o = __shfl_xor(most, d);
      most = o > most ? o : most;
    }
    const bool finite = most < 0x7f800000u;
    constexpr bool kHalf = sizeof(Elem) == 2 && T::kPer16 == 8 && __is_same(T, TypeF16);
    if (kHalf && finite && most > __float_as_uint(kLargestHalf)) most = __float_as_uint(kLargestHalf);
    int e = (int)(most >> 23) - 135 + ((most & 0x7fffffu) > 0x600000u);
    e = most == 0 || !finite ? 0 : e < kLeastPower ? kLeastPower : e;
    if (there) {
      const float f = __uint_as_float((uint32_t)(127 - e) << 23);
      u32x2 c;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[k] = v[4 * j + k];
          if (kHalf) y[k] = fminf(fmaxf(y[k], -kLargestHalf), kLargestHalf);
          y[k] *= f;
        }
        c[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
      }
      if (!finite) c = u32x2(0x7f7f7f7fu);
      *(u32x2*)code = c;
      if (col == 0) *scale = (uint8_t)(e + 127);
    }
  }
}

template <class T>
void launch_typed(const CacheRows& a, bool read, hipStream_t st) {
  const uint64_t rows = 2 * (uint64_t)a.batch * a.length * a.heads;
  const uint32_t grid = (uint32_t)((rows + 256 / kRowLanes - 1) / (256 / kRowLanes));
  if (read) cache_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else cache_kernel<T, false><<<grid, 256, 0, st>>>(a);
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
