// C ABI of candidates and answers that share a prompt (declared in
// include/dizo_amd.h): argument checks, then one or two launches.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "../../include/dizo_amd.h"
#include "dz_common.h"
#include "dz_internal.h"
#include "dz_prefix.h"
#include "dz_sampling.h"

namespace {

using dz::api_fail;

constexpr int64_t kMaxDim = (int64_t)1 << 24;      // of one dimension
constexpr int64_t kMaxRows = (int64_t)1 << 31;     // queries, or rows of a cache call: 32-bit grids and row numbers
constexpr int64_t kMaxStride = (int64_t)1 << 52;   // elements
constexpr int64_t kMaxSlotStride = (int64_t)1 << 24;  // a tile's offsets are 32-bit

int32_t invalid(const std::string& msg) { return api_fail(DZ_ERR_INVALID, msg); }

int32_t check_dtype(int32_t dtype) {
  if (dtype != DZ_DTYPE_F32 && dtype != DZ_DTYPE_F16 && dtype != DZ_DTYPE_BF16) return invalid("unknown dtype code " + std::to_string(dtype));
  return DZ_OK;
}
int64_t size_of(int32_t dtype) { return dtype == DZ_DTYPE_F32 ? 4 : 2; }

int32_t check_dim(int64_t x, int64_t least, const char* what) {
  if (x < least || x > kMaxDim) return invalid(std::string(what) + " out of range: " + std::to_string(x));
  return DZ_OK;
}

// A tensor of four strided dimensions of rows of `inner` elements; [first, first + bytes) holds all of it.
struct Extent {
  uint64_t first, end;
};
int32_t check_tensor(const void* p, int64_t es, const int64_t (&dims)[4], const int64_t* strides, int64_t inner, int64_t align,
                     const char* what, Extent* extent) {
  if (!p) return invalid(std::string(what) + " is NULL");
  if ((uintptr_t)p % (uintptr_t)align) return invalid(std::string(what) + " is not aligned to " + std::to_string(align) + " bytes");
  int64_t n = inner;
  for (int i = 0; i < 4; ++i) {
    if (dims[i] == 1) continue;  // the stride is not used
    if (strides[i] < 0) return invalid(std::string(what) + ": negative stride");
    if (strides[i] > kMaxStride / dims[i]) return invalid(std::string(what) + ": stride out of range");
    if (strides[i] * es % align) return invalid(std::string(what) + ": a stride is not a multiple of " + std::to_string(align) + " bytes");
    n += (dims[i] - 1) * strides[i];
  }
  if (extent) *extent = {(uint64_t)(uintptr_t)p, (uint64_t)(uintptr_t)p + (uint64_t)(n * es)};
  return dz::api_check_range(p, (uint64_t)n * (uint64_t)es, what);
}

// Rows that are written do not share elements: sorted by stride, each dimension steps over the ones below it.
int32_t check_distinct(const int64_t (&dims)[4], const int64_t* strides, int64_t inner, const char* what) {
  int order[4] = {0, 1, 2, 3};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (strides[order[j]] < strides[order[i]]) {
        const int t = order[i];
        order[i] = order[j];
        order[j] = t;
      }
  int64_t span = inner;
  for (int i = 0; i < 4; ++i) {
    const int d = order[i];
    if (dims[d] == 1) continue;
    if (strides[d] < span) return invalid(std::string(what) + ": rows overlap");
    span += (dims[d] - 1) * strides[d];
  }
  return DZ_OK;
}

bool overlap(const Extent& a, const Extent& b) { return a.first < b.end && b.first < a.end; }

// Whether two tensors of the same dimensions, by strides in bytes, share none. They lie apart, or their outer dimensions have the same
// strides, and what lies inside of these is apart and fits into the least of them: rows of keys and values in turn, or
// codes with their scales behind them.
bool apart(const int64_t (&dims)[4], const Extent& a, const int64_t* a_strides, const Extent& b, const int64_t* b_strides) {
  if (!overlap(a, b)) return true;
  int order[4], n = 0;  // the largest stride first, dimensions of one element aside
  for (int i = 0; i < 4; ++i) {
    if (dims[i] == 1) continue;
    int at = n++;
    for (; at > 0 && a_strides[order[at - 1]] < a_strides[i]; --at) order[at] = order[at - 1];
    order[at] = i;
  }
  int64_t a_size = (int64_t)(a.end - a.first), b_size = (int64_t)(b.end - b.first);
  const int64_t off = (int64_t)(b.first - a.first);
  for (int outer = 0; outer < n; ++outer) {
    const int64_t stride = a_strides[order[outer]], steps = dims[order[outer]] - 1;
    if (b_strides[order[outer]] != stride) return false;
    a_size -= steps * stride;
    b_size -= steps * stride;
    if (off < a_size && -off < b_size) continue;
    int64_t span = (off + b_size > a_size ? off + b_size : a_size) - (off < 0 ? off : 0);
    bool fits = true;
    for (int i = outer; i >= 0 && fits; --i) {
      fits = a_strides[order[i]] >= span;
      span += (dims[order[i]] - 1) * a_strides[order[i]];
    }
    if (fits) return true;
  }
  return false;
}

#define DZ_TRY(expr)             \
  do {                           \
    const int32_t rc_ = (expr);  \
    if (rc_) return rc_;         \
  } while (0)

int32_t check_store(const dz_keys_values& kv, int32_t dtype, bool bytes, const int64_t (&dims)[4], int64_t width, const std::string& name,
                    Extent* extents) {
  const int64_t es = bytes ? 1 : size_of(dtype), align = bytes ? 8 : 16;
  DZ_TRY(check_tensor(kv.k, es, dims, kv.k_strides, width, align, (name + " keys").c_str(), extents));
  DZ_TRY(check_tensor(kv.v, es, dims, kv.v_strides, width, align, (name + " values").c_str(), extents + 1));
  if (dims[3] > 1 && (kv.k_strides[3] >= kMaxSlotStride || kv.v_strides[3] >= kMaxSlotStride))
    return invalid(name + ": slots are " + std::to_string(kMaxSlotStride) + " elements or more apart");
  if (bytes) {
    DZ_TRY(check_tensor(kv.k_scales, 1, dims, kv.k_scale_strides, 1, 1, (name + " key scales").c_str(), extents + 2));
    DZ_TRY(check_tensor(kv.v_scales, 1, dims, kv.v_scale_strides, 1, 1, (name + " value scales").c_str(), extents + 3));
    if (dims[3] > 1 && (kv.k_scale_strides[3] >= kMaxSlotStride || kv.v_scale_strides[3] >= kMaxSlotStride))
      return invalid(name + " scales: slots are " + std::to_string(kMaxSlotStride) + " bytes or more apart");
  }
  return DZ_OK;
}

void copy4(int64_t* to, const int64_t* from) {
  for (int i = 0; i < 4; ++i) to[i] = from[i];
}

dz::KeyValues store_of(const dz_keys_values& x) {
  dz::KeyValues kv{};
  kv.k = x.k;
  kv.v = x.v;
  copy4(kv.k_s, x.k_strides);
  copy4(kv.v_s, x.v_strides);
  kv.k_scale = x.k_scales;
  kv.v_scale = x.v_scales;
  copy4(kv.k_scale_s, x.k_scale_strides);
  copy4(kv.v_scale_s, x.v_scale_strides);
  return kv;
}

// The sizes of a call, and what they plan. No pointer is looked at but for NULL scales.
int32_t plan_of(const dz_attention* x, dz::Attend* a, dz::AttendPlan* plan) {
  if (!x) return invalid("a is NULL");
  DZ_TRY(check_dtype(x->dtype));
  DZ_TRY(check_dim(x->groups, 0, "groups"));
  DZ_TRY(check_dim(x->sequences, 0, "sequences"));
  DZ_TRY(check_dim(x->heads, 1, "heads"));
  DZ_TRY(check_dim(x->kv_heads, 1, "kv_heads"));
  DZ_TRY(check_dim(x->length, 0, "length"));
  DZ_TRY(check_dim(x->slots, 0, "slots"));
  DZ_TRY(check_dim(x->prefix_slots, 0, "prefix_slots"));
  if (x->heads % x->kv_heads) return invalid("heads (" + std::to_string(x->heads) + ") is not a multiple of kv_heads (" + std::to_string(x->kv_heads) + ")");
  if (x->width < 8 || x->width > 128 || x->width % 8) return invalid("width must be a multiple of 8 up to 128, got " + std::to_string(x->width));
  if (!(x->scale > 0.f && x->scale <= 0x1p126f)) return invalid("scale must be positive, 2^126 at most");  // (with log2 e it is finite)
  int64_t rows = 1;
  for (int64_t d : {x->groups, x->sequences, x->heads, x->length}) {
    if (d && rows > kMaxRows / d) return invalid("too many queries: " + std::to_string(kMaxRows) + " at most");
    rows *= d;
  }
  if (rows >= kMaxRows) return invalid("too many queries: " + std::to_string(kMaxRows) + " at most");
  if (!x->slots && !x->prefix_slots) return invalid("neither own keys nor a prefix");
  const bool own = x->slots > 0, prefix = x->prefix_slots > 0;
  const bool own_bytes = own && x->own.k_scales, prefix_bytes = prefix && x->prefix.k_scales;
  if (own && prefix && own_bytes != prefix_bytes) return invalid("one of own and prefix is an 8-bit store and the other is not");
  a->groups = (int32_t)x->groups;
  a->sequences = (int32_t)x->sequences;
  a->heads = (int32_t)x->heads;
  a->kv_heads = (int32_t)x->kv_heads;
  a->length = (int32_t)x->length;
  a->width = (int32_t)x->width;
  a->slots = (int32_t)x->slots;
  a->prefix_slots = (int32_t)x->prefix_slots;
  a->bytes = own_bytes || prefix_bytes;
  a->scale = x->scale;
  if (!rows) {
    *plan = {};
    return DZ_OK;
  }
  *plan = dz::attend_plan(x->dtype, *a);
  if (plan->items > 1 << 22) return invalid("too many tiles of queries");  // a launch counts its threads in 32 bits
  return DZ_OK;
}

// Whether an 8-bit store's rows start at multiples of 16 bytes.
bool in_chunks(const dz_keys_values& kv) {
  uint64_t low = (uint64_t)(uintptr_t)kv.k | (uint64_t)(uintptr_t)kv.v;
  for (int i = 0; i < 4; ++i) low |= (uint64_t)kv.k_strides[i] | (uint64_t)kv.v_strides[i];
  return low % 16 == 0;
}

int32_t launched(hipError_t e, const char* what) { return e == hipSuccess ? DZ_OK : dz::api_hip_fail(e, what); }

int32_t cache_call(const dz_keys_values* kv, const dz_keys_values* cache, int32_t dtype, int64_t batch, int64_t heads, int64_t length,
                   int64_t width, int64_t slots, const int32_t* positions, int64_t position, bool read, void* stream) {
  DZ_TRY(check_dtype(dtype));
  if (!kv || !cache) return invalid("kv or cache is NULL");
  DZ_TRY(check_dim(batch, 0, "batch"));
  DZ_TRY(check_dim(heads, 1, "heads"));
  DZ_TRY(check_dim(length, 0, "length"));
  DZ_TRY(check_dim(slots, 1, "slots"));
  if (width < 8 || width > 128 || width % 8) return invalid("width must be a multiple of 8 up to 128, got " + std::to_string(width));
  int64_t rows = 1;
  for (int64_t d : {batch, heads, length}) {
    if (d && rows > (kMaxRows >> 4) / d) return invalid("too many rows");  // 16 lanes each, counted in 32 bits with both stores
    rows *= d;
  }
  if (rows >= (kMaxRows >> 4)) return invalid("too many rows");
  if (!positions && (position < 0 || position > slots - length))
    return invalid("tokens " + std::to_string(position) + " to " + std::to_string(position + length) + " do not fit " + std::to_string(slots) + " slots");
  if (!rows) return DZ_OK;
  const int64_t es = size_of(dtype), in_dims[4] = {batch, 1, heads, length}, dims[4] = {batch, 1, heads, slots};
  Extent x[2], c[4], at{};
  DZ_TRY(check_tensor(kv->k, es, in_dims, kv->k_strides, width, 16, "k", x));
  DZ_TRY(check_tensor(kv->v, es, in_dims, kv->v_strides, width, 16, "v", x + 1));
  if (!cache->k_scales || !cache->v_scales) return invalid("cache scales are NULL");
  DZ_TRY(check_store(*cache, dtype, true, dims, width, "cache", c));
  if (positions) {
    const int64_t all[4] = {1, 1, 1, batch}, dense[4] = {0, 0, 0, 1};
    DZ_TRY(check_tensor(positions, 4, all, dense, 1, 4, "positions", &at));
    for (const Extent& f : c)
      if (overlap(at, f)) return invalid("the cache overlaps positions");
  }
  if (read) {
    DZ_TRY(check_distinct(in_dims, kv->k_strides, width, "k"));
    DZ_TRY(check_distinct(in_dims, kv->v_strides, width, "v"));
    if (overlap(x[0], x[1])) return invalid("k and v overlap");
  } else {
    DZ_TRY(check_distinct(dims, cache->k_strides, width, "cache keys"));
    DZ_TRY(check_distinct(dims, cache->v_strides, width, "cache values"));
    DZ_TRY(check_distinct(dims, cache->k_scale_strides, 1, "cache key scales"));
    DZ_TRY(check_distinct(dims, cache->v_scale_strides, 1, "cache value scales"));
    const int64_t* const strides[4] = {cache->k_strides, cache->v_strides, cache->k_scale_strides, cache->v_scale_strides};
    for (int i = 0; i < 4; ++i)
      for (int j = i + 1; j < 4; ++j)
        if (!apart(dims, c[i], strides[i], c[j], strides[j])) return invalid("the cache's keys, values or scales overlap");
  }
  for (const Extent& e : x)
    for (const Extent& f : c)
      if (overlap(e, f)) return invalid("the cache overlaps k or v");
  dz::CacheRows a{};
  for (int i = 0; i < 2; ++i) {
    const int64_t* xs = i ? kv->v_strides : kv->k_strides;
    const int64_t* cs = i ? cache->v_strides : cache->k_strides;
    const int64_t* ss = i ? cache->v_scale_strides : cache->k_scale_strides;
    a.x[i] = i ? kv->v : kv->k;
    a.code[i] = const_cast<void*>(i ? cache->v : cache->k);
    a.scale[i] = const_cast<uint8_t*>(i ? cache->v_scales : cache->k_scales);
    for (int d = 0; d < 3; ++d) {
      const int from = d ? d + 1 : 0;
      a.x_s[i][d] = xs[from];
      a.code_s[i][d] = cs[from];
      a.scale_s[i][d] = ss[from];
    }
  }
  a.positions = positions;
  a.position = (int32_t)position;
  a.batch = (int32_t)batch;
  a.heads = (int32_t)heads;
  a.length = (int32_t)length;
  a.width = (int32_t)width;
  a.slots = (int32_t)slots;
  return launched(dz::launch_cache(dtype, a, read, (hipStream_t)stream), read ? "cache_read kernel launch" : "cache_write kernel launch");
}

}  // namespace

extern "C" {

int32_t dz_shared_prefix_attention_workspace(const dz_attention* x, int64_t* bytes) {
  dz::Attend a{};
  dz::AttendPlan plan;
  DZ_TRY(plan_of(x, &a, &plan));
  if (!bytes) return invalid("bytes is NULL");
  *bytes = dz::attend_workspace(a, plan);
  return DZ_OK;
}

int32_t dz_shared_prefix_attention(const dz_attention* x, void* workspace, int64_t workspace_bytes, void* stream) {
  dz::Attend a{};
  dz::AttendPlan plan;
  DZ_TRY(plan_of(x, &a, &plan));
  if (!x->groups || !x->sequences || !x->length) return DZ_OK;
  const int64_t es = size_of(x->dtype), rows[4] = {x->groups, x->sequences, x->heads, x->length};
  Extent q, out, in[8] = {};
  DZ_TRY(check_tensor(x->q, es, rows, x->q_strides, x->width, 16, "q", &q));
  DZ_TRY(check_tensor(x->out, es, rows, x->out_strides, x->width, 16, "out", &out));
  DZ_TRY(check_distinct(rows, x->out_strides, x->width, "out"));
  if (x->slots) {
    const int64_t dims[4] = {x->groups, x->sequences, x->kv_heads, x->slots};
    DZ_TRY(check_store(x->own, x->dtype, a.bytes, dims, x->width, "own", in));
  }
  if (x->prefix_slots) {
    const int64_t dims[4] = {x->groups, 1, x->kv_heads, x->prefix_slots};
    DZ_TRY(check_store(x->prefix, x->dtype, a.bytes, dims, x->width, "prefix", in + 4));
  }
  if (overlap(out, q)) return invalid("out and q overlap");
  for (const Extent& e : in)
    if (overlap(out, e)) return invalid("out overlaps keys or values");
  const int64_t dense[4] = {0, 0, 0, 1};
  if (x->positions) {
    const int64_t n[4] = {1, 1, 1, x->groups * x->sequences};
    Extent at;
    DZ_TRY(check_tensor(x->positions, 4, n, dense, 1, 4, "positions", &at));
    if (overlap(out, at)) return invalid("out overlaps positions");
  }
  if (x->prefix_lengths) {
    const int64_t n[4] = {1, 1, 1, x->groups};
    Extent at;
    DZ_TRY(check_tensor(x->prefix_lengths, 4, n, dense, 1, 4, "prefix_lengths", &at));
    if (overlap(out, at)) return invalid("out overlaps prefix_lengths");
  }
  const int64_t need = dz::attend_workspace(a, plan);
  if (workspace_bytes < need)
    return invalid("workspace of " + std::to_string(workspace_bytes) + " bytes: " + std::to_string(need) + " are needed");
  if (need) {
    const int64_t n[4] = {1, 1, 1, (need + 15) / 16};
    Extent work;
    DZ_TRY(check_tensor(workspace, 16, n, dense, 1, 16, "workspace", &work));
    if (overlap(work, q) || overlap(work, out)) return invalid("workspace overlaps q or out");
    for (const Extent& e : in)
      if (overlap(work, e)) return invalid("workspace overlaps keys or values");
  }
  a.q = x->q;
  a.out = x->out;
  copy4(a.q_s, x->q_strides);
  copy4(a.out_s, x->out_strides);
  a.own = store_of(x->own);
  a.prefix = store_of(x->prefix);
  a.whole_chunks = a.bytes && x->width % 16 == 0 && (!x->slots || in_chunks(x->own)) && (!x->prefix_slots || in_chunks(x->prefix));
  a.positions = x->positions;
  a.prefix_lengths = x->prefix_lengths;
  return launched(dz::launch_attend(x->dtype, a, plan, workspace, (hipStream_t)stream), "shared_prefix_attention kernel launch");
}

int32_t dz_cache_write(const dz_keys_values* kv, const dz_keys_values* cache, int32_t dtype, int64_t batch, int64_t heads, int64_t length,
                       int64_t width, int64_t slots, const int32_t* positions, int64_t position, void* stream) {
  return cache_call(kv, cache, dtype, batch, heads, length, width, slots, positions, position, false, stream);
}

int32_t dz_cache_read(const dz_keys_values* cache, const dz_keys_values* kv, int32_t dtype, int64_t batch, int64_t heads, int64_t length,
                      int64_t width, int64_t slots, int64_t position, void* stream) {
  return cache_call(kv, cache, dtype, batch, heads, length, width, slots, nullptr, position, true, stream);
}

int32_t dz_sample_tokens(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t logits_stride, const float* uniform,
                         double temperature, int32_t top_k, double top_p, double min_p, const float* temperatures, const int32_t* top_ks,
                         const float* top_ps, const float* min_ps, int64_t* tokens, void* stream) {
  DZ_TRY(check_dtype(dtype));
  if (rows < 0 || rows >= (1 << 22)) return invalid("row count out of range: " + std::to_string(rows) + " (at most 4194303 rows)");
  if (vocab < 1 || vocab > (int64_t)dz::kMaxSampleVocab)
    return invalid("vocab out of range: " + std::to_string(vocab) + " (at most " + std::to_string(dz::kMaxSampleVocab) + ")");
  if (!temperatures && temperature != 0 && !(temperature >= 0x1p-63 && temperature < 0x1p64))
    return invalid("temperature must be 0, or from 2^-63 up to 2^64");
  if (!top_ks && top_k < 0) return invalid("top_k must not be negative");
  if (!top_ps && !(top_p >= 0 && top_p <= 1)) return invalid("top_p must be 0 to 1");
  if (!min_ps && !(min_p >= 0 && min_p <= 1)) return invalid("min_p must be 0 to 1");
  if (!rows) return DZ_OK;
  const int64_t es = size_of(dtype), n[4] = {1, 1, 1, rows}, dense[4] = {0, 0, 0, 1}, strides[4] = {0, 0, 0, logits_stride};
  const struct {
    const void* p;
    const char* what;
  } of_row[] = {{uniform, "uniform"}, {temperatures, "temperatures"}, {top_ks, "top_ks"}, {top_ps, "top_ps"}, {min_ps, "min_ps"}};
  Extent in[6] = {}, out;
  DZ_TRY(check_tensor(logits, es, n, strides, vocab, es, "logits", in + 5));
  for (int i = 0; i < 5; ++i)
    if (i == 0 || of_row[i].p) DZ_TRY(check_tensor(of_row[i].p, 4, n, dense, 1, 4, of_row[i].what, in + i));
  DZ_TRY(check_tensor(tokens, 8, n, dense, 1, 8, "tokens", &out));
  for (const Extent& e : in)
    if (overlap(out, e)) return invalid("tokens overlap an input");
  dz::SampleRows a{};
  a.logits = logits;
  a.stride = logits_stride;
  a.nrows = (uint32_t)rows;
  a.vocab = (uint32_t)vocab;
  a.uniform = uniform;
  a.temperatures = temperatures;
  a.top_ks = top_ks;
  a.top_ps = top_ps;
  a.min_ps = min_ps;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.tokens = tokens;
  return launched(dz::launch_sample(dtype, a, (hipStream_t)stream), "sample_tokens kernel launch");
}

}  // extern "C"
