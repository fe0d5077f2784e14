// Log probabilities and entropies straight from hidden states and the
// language-model head: the products are reduced to softmax statistics where
// they are made, and the logits are never stored.
#include "dz_token_loss.h"
#include "dz_token_math.h"

namespace dz {
namespace {

// 16 bytes of a row's width per lane: lane l holds row l & 15, bytes
// 16 (l >> 4) .. + 15 of a 64-byte slab. The products of one slab: 16 head
// rows by 16 tokens; lane l then holds token l & 15, head rows 4 (l >> 4) .. + 3.
template <class T>
struct Frag;
template <>
struct Frag<TypeF16> {
  using V = TypeF16::V;
  __device__ static f32x4 mma(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<TypeBF16> {
  using V = TypeBF16::V;
  __device__ static f32x4 mma(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<TypeF32> {
  using V = TypeF32::V;
  // the slab's 16 columns in the order (0, 4, 8, 12), (1, 5, ...), the same on both sides
  __device__ static f32x4 mma(V a, V b, f32x4 c) {
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

struct Work {
  uint32_t* count;   // live rows
  uint32_t* row_of;  // live row -> row
  uint32_t* live_of;  // row -> live row
  float* token_logit;  // per live row
  float4* partial;     // (live row, head tile)
};
constexpr uint32_t kTile = 64;  // head rows of a workgroup

__host__ __device__ inline uint64_t align256(uint64_t x) { return (x + 255) / 256 * 256; }
inline uint32_t head_tiles(uint32_t vocab) { return (vocab + kTile - 1) / kTile; }
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

// 16 bytes from column `col` of a row; columns past the width are 0.
template <class T>
__device__ typename Frag<T>::V load16(const typename T::Elem* row, uint32_t col, uint32_t width, bool vec) {
  if (vec && col + T::kPer16 <= width) return *(const typename Frag<T>::V*)(row + col);
  typename T::V v;
  for (int j = 0; j < T::kPer16; ++j) v[j] = col + j < width ? row[col + j] : (typename T::Elem)0.f;
  return v;
}

template <class T>
__global__ __launch_bounds__(256) void head_kernel(HeadRows a, Work w, uint32_t tiles, bool vec) {
  __shared__ SoftStats sh[4][16];
  const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, count = *w.count;
  const uint32_t at = blockIdx.y * 16 + (lane & 15);
  if (blockIdx.y * 16 >= count) return;
  const uint32_t row = w.row_of[at < count ? at : count - 1];
  const uint32_t v0 = blockIdx.x * kTile + wv * 16;
  const uint32_t vr = v0 + (lane & 15) < a.vocab ? v0 + (lane & 15) : a.vocab - 1;
  const typename T::Elem* h = (const typename T::Elem*)a.hidden + (int64_t)row * a.hidden_stride;
  const typename T::Elem* e = (const typename T::Elem*)a.weight + (int64_t)vr * a.weight_stride;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const uint32_t lane_col = (lane >> 4) * T::kPer16;
  for (uint32_t k = 0; k < a.width; k += 4 * T::kPer16)  // the same trips for the whole wave
    acc = Frag<T>::mma(load16<T>(e, k + lane_col, a.width, vec), load16<T>(h, k + lane_col, a.width, vec), acc);
  const int64_t tok = a.tokens[row];
  SoftStats st = SoftStats::of(-INFINITY);
  for (int j = 0; j < 4; ++j)
    if (v0 + 4 * (lane >> 4) + j < a.vocab) st.m = fmaxf(st.m, acc[j]);
  for (int j = 0; j < 4; ++j) {
    const uint32_t v = v0 + 4 * (lane >> 4) + j;
    if (v >= a.vocab) continue;
    st.add(acc[j], kLog2e);
    if ((int64_t)v == tok && at < count) w.token_logit[at] = acc[j];
  }
  for (int off = 16; off <= 32; off *= 2) {
    SoftStats o;
    o.m = __shfl_xor(st.m, off, 64);
    o.s = __shfl_xor(st.s, off, 64);
    o.t = __shfl_xor(st.t, off, 64);
    st.join(o, kLog2e);
  }
  if (lane < 16) sh[wv][lane] = st;
  __syncthreads();
  if (wv == 0 && lane < 16 && at < count) {
    for (int i = 1; i < 4; ++i) st.join(sh[i][lane], kLog2e);
    w.partial[(uint64_t)at * tiles + blockIdx.x] = float4{st.m, st.s, st.t, 0.f};
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
  const uint32_t at = w.live_of[r];
  SoftStats st = SoftStats::of(-INFINITY);
  for (uint32_t i = lane; i < tiles; i += 64) {
    const float4 p = w.partial[(uint64_t)at * tiles + i];
    SoftStats o;
    o.m = p.x;
    o.s = p.y;
    o.t = p.z;
    st.join(o, kLog2e);
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
    a.logprobs[r] = valid && inside ? st.lnq(w.token_logit[at], 1.f) : NAN;
    a.entropy[r] = valid ? kLn2 * (log2s - st.t / st.s) : NAN;
  }
}

}  // namespace

int64_t head_workspace(int dtype, uint32_t nrows, uint32_t width, uint32_t vocab) {
  (void)dtype;
  (void)width;
  return (int64_t)(256 + 3 * align256((uint64_t)nrows * 4) + (uint64_t)nrows * head_tiles(vocab) * sizeof(float4));
}

hipError_t launch_head(int dtype, const HeadRows& a, void* workspace, hipStream_t st) {
  const Work w = work_of(workspace, a.nrows);
  const uint32_t tiles = head_tiles(a.vocab);
  const int64_t es = dtype == DZ_F32 ? 4 : 2;
  const bool vec = ((uint64_t)a.hidden | (uint64_t)a.weight | (uint64_t)(a.hidden_stride * es) |
                    (uint64_t)(a.weight_stride * es)) % 16 == 0;
  live_rows_kernel<<<1, 1024, 0, st>>>(a, w);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(tiles, (a.nrows + 15) / 16);
  if (dtype == DZ_F32) head_kernel<TypeF32><<<grid, 256, 0, st>>>(a, w, tiles, vec);
  else if (dtype == DZ_F16) head_kernel<TypeF16><<<grid, 256, 0, st>>>(a, w, tiles, vec);
  else head_kernel<TypeBF16><<<grid, 256, 0, st>>>(a, w, tiles, vec);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  head_join_kernel<<<a.nrows, 64, 0, st>>>(a, w, tiles);
  return hipGetLastError();
}

}  // namespace dz
