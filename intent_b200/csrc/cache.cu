// Writing rows of keys and values into a paged cache and reading them back, in 16 or 8 bits.
//
// Both directions are bound by HBM: 2 bytes an element on the rows' side, 1 or 2 on the cache's and
// 4 for a row's scale.  A row of D columns belongs to D / 16 lanes of a warp (rounded up to a power
// of two), 16 columns a lane: two 128-bit vectors of rows against one of codes (two in 16 bits), the
// row's largest magnitude by a butterfly over those lanes.  One launch moves keys and values: a unit
// is the key row and the value row of ROWS heads of a token, all of whose loads are in flight
// together, and shares one look at the slot and one division by the page size.
#include "cache.cuh"

namespace b200 {
namespace {

using cache::Cache;
using heads::Eight;
using heads::View3;
using heads::View4;

constexpr int kThreads = 256;

struct Rows {                // (tokens, heads, columns)
  void *k, *v;
  int64_t k_token, k_head, v_token, v_head;
};
struct Pages {               // (pages, heads, page_size, columns), scales (pages, heads, page_size)
  void *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  float *k_scale, *v_scale;
  int64_t ks_page, ks_head, ks_slot, vs_page, vs_head, vs_slot;
};
struct Extents {
  const int64_t *slots;
  int64_t slots_step, capacity;
  int tokens, heads, columns, page_size, slices, store;
  int *status;
};

// Slot of a token, or -1 where there is none (padding; a slot behind the cache, which is reported).
__device__ __forceinline__ int64_t slot_of(const Extents &x, int token, bool first_lane) {
  const int64_t slot = x.slots[token * x.slots_step];
  if (slot < x.capacity) return slot < 0 ? -1 : slot;
  if (first_lane) heads::report_index(x.status, token);
  return -1;
}

template <typename T> __device__ __forceinline__ uint32_t magnitude(const Eight<T> &a, const Eight<T> &b) {
  const uint32_t words[8] = {a.raw[0].x, a.raw[0].y, a.raw[0].z, a.raw[0].w, b.raw[0].x, b.raw[0].y, b.raw[0].z, b.raw[0].w};
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = __vmaxu2(most, words[i] & 0x7fff7fffu);   // 16-bit floats of one sign order as their bits
  return max(most & 0xffffu, most >> 16);
}

template <typename T, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(Rows rows, Pages pages, Extents x) {
  const int e = threadIdx.x % LANES;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / x.slices);
  const int head0 = (int)(unit - (int64_t)token * x.slices) * ROWS;
  const int64_t slot = token < x.tokens ? slot_of(x, token, e == 0) : -1;
  const bool lane_live = token < x.tokens && e * 16 < x.columns;
  Eight<T> a[2 * ROWS], b[2 * ROWS];   // keys, then values
  const T *k = static_cast<const T *>(rows.k) + (lane_live ? token * rows.k_token + e * 16 : 0);
  const T *v = static_cast<const T *>(rows.v) + (lane_live ? token * rows.v_token + e * 16 : 0);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int head = head0 + i;
    a[i].clear(); b[i].clear(); a[ROWS + i].clear(); b[ROWS + i].clear();
    if (lane_live && head < x.heads) {
      a[i].load(k + head * rows.k_head);
      b[i].load(k + head * rows.k_head + 8);
      a[ROWS + i].load(v + head * rows.v_head);
      b[ROWS + i].load(v + head * rows.v_head + 8);
    }
  }
  int64_t page = 0;
  int offset = 0;
  if (slot >= 0) cache::locate(slot, x.page_size, page, offset);
#pragma unroll
  for (int i = 0; i < 2 * ROWS; ++i) {
    const bool is_key = i < ROWS;
    const int head = head0 + (is_key ? i : i - ROWS);
    const bool live = lane_live && slot >= 0 && head < x.heads;
    const int64_t to = is_key ? page * pages.k_page + head * pages.k_head + offset * pages.k_slot
                              : page * pages.v_page + head * pages.v_head + offset * pages.v_slot;
    void *base = is_key ? pages.k : pages.v;
    if (x.store == cache::kNative) {
      if (live) {
        a[i].store(static_cast<T *>(base) + to + e * 16);
        b[i].store(static_cast<T *>(base) + to + e * 16 + 8);
      }
      continue;
    }
    uint32_t most = magnitude(a[i], b[i]);
#pragma unroll
    for (int offset_lane = LANES / 2; offset_lane > 0; offset_lane >>= 1)
      most = max(most, __shfl_xor_sync(0xffffffffu, most, offset_lane));
    const uint16_t bits = (uint16_t)most;
    const uint32_t wide = __float_as_uint(Element<T>::widen(*reinterpret_cast<const T *>(&bits)));
    const float scale = x.store == cache::kInt8 ? cache::int8_scale(wide) : cache::e4m3_scale(wide);
    if (live) {
      float values[16];
      a[i].widen(values);
      b[i].widen(values + 8);
      *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(base) + to + e * 16) = cache::encode(values, x.store, scale);
      if (e == 0)
        *(is_key ? pages.k_scale + page * pages.ks_page + head * pages.ks_head + offset * pages.ks_slot
                 : pages.v_scale + page * pages.vs_page + head * pages.vs_head + offset * pages.vs_slot) = scale;
    }
  }
}

template <typename T, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(Rows rows, Pages pages, Extents x) {
  const int e = threadIdx.x % LANES;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / x.slices);
  const int head0 = (int)(unit - (int64_t)token * x.slices) * ROWS;
  const bool lane_live = token < x.tokens && e * 16 < x.columns;
  if (!lane_live) return;
  const int64_t slot = slot_of(x, token, e == 0);
  int64_t page = 0;
  int offset = 0;
  if (slot >= 0) cache::locate(slot, x.page_size, page, offset);
  uint4 codes[2 * ROWS];
  float scale[2 * ROWS];
#pragma unroll
  for (int i = 0; i < 2 * ROWS; ++i) {
    const bool is_key = i < ROWS;
    const int head = head0 + (is_key ? i : i - ROWS);
    codes[i] = make_uint4(0, 0, 0, 0);
    scale[i] = 0.0f;
    if (slot < 0 || head >= x.heads) continue;
    const int64_t from = is_key ? page * pages.k_page + head * pages.k_head + offset * pages.k_slot
                                : page * pages.v_page + head * pages.v_head + offset * pages.v_slot;
    codes[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(is_key ? pages.k : pages.v) + from + e * 16);
    scale[i] = is_key ? pages.k_scale[page * pages.ks_page + head * pages.ks_head + offset * pages.ks_slot]
                      : pages.v_scale[page * pages.vs_page + head * pages.vs_head + offset * pages.vs_slot];
  }
#pragma unroll
  for (int i = 0; i < 2 * ROWS; ++i) {
    const bool is_key = i < ROWS;
    const int head = head0 + (is_key ? i : i - ROWS);
    if (head >= x.heads) continue;
    float values[16];
    cache::decode(codes[i], x.store, scale[i], values);
    Eight<T> a, b;
    a.narrow(values);
    b.narrow(values + 8);
    T *to = static_cast<T *>(is_key ? rows.k : rows.v) + e * 16 +
            (is_key ? token * rows.k_token + head * rows.k_head : token * rows.v_token + head * rows.v_head);
    a.store(to);
    b.store(to + 8);
  }
}

// A 16-bit cache gives its rows back as they are (16 columns a lane, two vectors).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads)
cache_read_native_kernel(Rows rows, Pages pages, Extents x) {
  const int e = threadIdx.x % LANES;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / x.heads);
  const int head = (int)(unit - (int64_t)token * x.heads);
  if (token >= x.tokens || e * 16 >= x.columns) return;
  const int64_t slot = slot_of(x, token, e == 0);
  Eight<T> k0, k1, v0, v1;
  k0.clear(); k1.clear(); v0.clear(); v1.clear();
  if (slot >= 0) {
    int64_t page;
    int offset;
    cache::locate(slot, x.page_size, page, offset);
    const T *k = static_cast<const T *>(pages.k) + page * pages.k_page + head * pages.k_head + offset * pages.k_slot + e * 16;
    const T *v = static_cast<const T *>(pages.v) + page * pages.v_page + head * pages.v_head + offset * pages.v_slot + e * 16;
    k0.load(k);
    k1.load(k + 8);
    v0.load(v);
    v1.load(v + 8);
  }
  T *k = static_cast<T *>(rows.k) + token * rows.k_token + head * rows.k_head + e * 16;
  T *v = static_cast<T *>(rows.v) + token * rows.v_token + head * rows.v_head + e * 16;
  k0.store(k);
  k1.store(k + 8);
  v0.store(v);
  v1.store(v + 8);
}

// --------------------------------------------------------------------- host
struct Arguments {
  View3 k, v;
  const void *slots;
  int64_t slots_d0, slots_s0;
  Cache cache;
  void *workspace;
  int64_t ws_d0, ws_s0;
  int32_t dtype, store;
};

int check(const char *what, const Arguments &a, bool write) {
  if (a.dtype != B200_F16 && a.dtype != B200_BF16)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: rows are f16 or bf16", what);
  int status = cache::check(what, a.cache, a.dtype, a.store, 256);
  if (status != B200_OK) return status;
  const View4 &c = a.cache.k;
  if (!heads::sane(a.k) || !heads::sane(a.v) || !heads::sane(a.slots_d0, a.slots_s0))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (a.k.d0 != a.v.d0 || a.k.d0 != a.slots_d0) return fail(B200_ERR_INVALID_ARGUMENT, "%s: rows and slots differ in number", what);
  if (a.k.d1 != c.d1 || a.v.d1 != c.d1 || a.k.d2 != c.d3 || a.v.d2 != c.d3)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the rows' heads or columns are not the cache's", what);
  if (a.k.d0 >= (int64_t(1) << 31)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: 2^31 rows or more", what);
  if (!a.workspace || a.ws_d0 < B200_WORKSPACE_WORDS || a.ws_s0 != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the workspace needs %d contiguous int32 words", what, B200_WORKSPACE_WORDS);
  if (!a.k.d0 || !a.k.d1) return B200_OK;
  if (!a.k.data || !a.v.data || !a.slots) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(a.slots) & 7) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: slots are 8-byte aligned", what);
  if (!heads::vector_rows(a.k, 2) || !heads::vector_rows(a.v, 2))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  // what is written overlaps nothing: not itself, not the other output, not what is read
  const int wide = heads::element_size(a.store);
  const bool scaled = wide == 1;
  const heads::Span row_spans[] = {heads::span(a.k, 2), heads::span(a.v, 2)};
  const heads::Span cache_spans[] = {heads::span(a.cache.k, wide), heads::span(a.cache.v, wide),
                                     scaled ? heads::span(a.cache.k_scale, 4) : heads::Span{0, 0},
                                     scaled ? heads::span(a.cache.v_scale, 4) : heads::Span{0, 0}};
  const bool apart = write ? heads::distinct(a.cache.k) && heads::distinct(a.cache.v) && heads::apart(a.cache.k, a.cache.v, wide) &&
                                 (!scaled || (heads::distinct(a.cache.k_scale) && heads::distinct(a.cache.v_scale) &&
                                              heads::apart(a.cache.k_scale, a.cache.v_scale, 4)))
                           : heads::distinct(a.k) && heads::distinct(a.v) && heads::apart(a.k, a.v, 2);
  if (!apart) return fail(B200_ERR_INVALID_ARGUMENT, "%s: what is written overlaps itself", what);
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 4; ++j)
      if (heads::overlap(row_spans[i], cache_spans[j]))
        return fail(B200_ERR_INVALID_ARGUMENT, "%s: the rows and the cache overlap", what);
  return B200_OK;
}

void pack(const Arguments &a, int rows_of_unit, Rows &rows, Pages &pages, Extents &x) {
  rows = {const_cast<void *>(a.k.data), const_cast<void *>(a.v.data), a.k.s0, a.k.s1, a.v.s0, a.v.s1};
  const Cache &c = a.cache;
  pages = {const_cast<void *>(c.k.data), const_cast<void *>(c.v.data), c.k.s0, c.k.s1, c.k.s2, c.v.s0, c.v.s1, c.v.s2,
           static_cast<float *>(const_cast<void *>(c.k_scale.data)), static_cast<float *>(const_cast<void *>(c.v_scale.data)),
           c.k_scale.s0, c.k_scale.s1, c.k_scale.s2, c.v_scale.s0, c.v_scale.s1, c.v_scale.s2};
  x = {};
  x.slots = static_cast<const int64_t *>(a.slots);
  x.slots_step = a.slots_s0;
  x.capacity = c.k.d0 * c.k.d2;
  x.tokens = (int)a.k.d0;
  x.heads = (int)c.k.d1;
  x.columns = (int)c.k.d3;
  x.page_size = (int)c.k.d2;
  x.slices = (x.heads + rows_of_unit - 1) / rows_of_unit;
  x.store = a.store == B200_I8 ? cache::kInt8 : a.store == B200_E4M3 ? cache::kE4m3 : cache::kNative;
  x.status = static_cast<int *>(a.workspace);
}

enum Direction { kWrite, kRead, kReadNative };
template <Direction DIRECTION, typename T, int LANES, int ROWS>
int launch(const Arguments &a, cudaStream_t stream) {
  Rows rows;
  Pages pages;
  Extents x;
  pack(a, ROWS, rows, pages, x);
  const int64_t units = (int64_t)x.tokens * x.slices, per_block = kThreads / LANES;
  const int64_t blocks = (units + per_block - 1) / per_block;
  if (blocks >= (int64_t(1) << 31)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "cache: too many rows for one launch");
  if (DIRECTION == kWrite) cache_write_kernel<T, LANES, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(rows, pages, x);
  if (DIRECTION == kRead) cache_read_kernel<T, LANES, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(rows, pages, x);
  if (DIRECTION == kReadNative) cache_read_native_kernel<T, LANES><<<(unsigned)blocks, kThreads, 0, stream>>>(rows, pages, x);
  B200_CUDA_TRY(cudaGetLastError());
  return B200_OK;
}
template <Direction DIRECTION, typename T, int ROWS> int by_lanes(const Arguments &a, cudaStream_t stream) {
  switch (heads::row_lanes(a.cache.k.d3)) {
  case 1: return launch<DIRECTION, T, 1, ROWS>(a, stream);
  case 2: return launch<DIRECTION, T, 2, ROWS>(a, stream);
  case 4: return launch<DIRECTION, T, 4, ROWS>(a, stream);
  case 8: return launch<DIRECTION, T, 8, ROWS>(a, stream);
  default: return launch<DIRECTION, T, 16, ROWS>(a, stream);
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

#define VIEW3(name) \
  heads::View3 { name, name##_d0, name##_d1, name##_d2, name##_s0, name##_s1, name##_s2 }
#define VIEW4(name) \
  heads::View4 { name, name##_d0, name##_d1, name##_d2, name##_d3, name##_s0, name##_s1, name##_s2, name##_s3 }

extern "C" int b200_cache_write(
    const void *k, int64_t k_d0, int64_t k_d1, int64_t k_d2, int64_t k_s0, int64_t k_s1, int64_t k_s2,
    const void *v, int64_t v_d0, int64_t v_d1, int64_t v_d2, int64_t v_s0, int64_t v_s1, int64_t v_s2,
    const void *slots, int64_t slots_d0, int64_t slots_s0,
    void *k_cache, int64_t k_cache_d0, int64_t k_cache_d1, int64_t k_cache_d2, int64_t k_cache_d3,
    int64_t k_cache_s0, int64_t k_cache_s1, int64_t k_cache_s2, int64_t k_cache_s3,
    void *v_cache, int64_t v_cache_d0, int64_t v_cache_d1, int64_t v_cache_d2, int64_t v_cache_d3,
    int64_t v_cache_s0, int64_t v_cache_s1, int64_t v_cache_s2, int64_t v_cache_s3,
    void *k_scale, int64_t k_scale_d0, int64_t k_scale_d1, int64_t k_scale_d2, int64_t k_scale_s0, int64_t k_scale_s1, int64_t k_scale_s2,
    void *v_scale, int64_t v_scale_d0, int64_t v_scale_d1, int64_t v_scale_d2, int64_t v_scale_s0, int64_t v_scale_s1, int64_t v_scale_s2,
    void *workspace, int64_t ws_d0, int64_t ws_s0, int32_t dtype, int32_t store, void *stream) {
  const Arguments a{VIEW3(k), VIEW3(v), slots, slots_d0, slots_s0,
                    {VIEW4(k_cache), VIEW4(v_cache), VIEW3(k_scale), VIEW3(v_scale)},
                    workspace, ws_d0, ws_s0, dtype, store};
  const int status = check("cache_write", a, true);
  if (status != B200_OK) return status;
  if (!k_d0 || !k_d1) return B200_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B200_F16 ? by_lanes<kWrite, __half, 1>(a, s) : by_lanes<kWrite, __nv_bfloat16, 1>(a, s);
}

extern "C" int b200_cache_read(
    const void *k_cache, int64_t k_cache_d0, int64_t k_cache_d1, int64_t k_cache_d2, int64_t k_cache_d3,
    int64_t k_cache_s0, int64_t k_cache_s1, int64_t k_cache_s2, int64_t k_cache_s3,
    const void *v_cache, int64_t v_cache_d0, int64_t v_cache_d1, int64_t v_cache_d2, int64_t v_cache_d3,
    int64_t v_cache_s0, int64_t v_cache_s1, int64_t v_cache_s2, int64_t v_cache_s3,
    const void *slots, int64_t slots_d0, int64_t slots_s0,
    const void *k_scale, int64_t k_scale_d0, int64_t k_scale_d1, int64_t k_scale_d2, int64_t k_scale_s0, int64_t k_scale_s1, int64_t k_scale_s2,
    const void *v_scale, int64_t v_scale_d0, int64_t v_scale_d1, int64_t v_scale_d2, int64_t v_scale_s0, int64_t v_scale_s1, int64_t v_scale_s2,
    void *k, int64_t k_d0, int64_t k_d1, int64_t k_d2, int64_t k_s0, int64_t k_s1, int64_t k_s2,
    void *v, int64_t v_d0, int64_t v_d1, int64_t v_d2, int64_t v_s0, int64_t v_s1, int64_t v_s2,
    void *workspace, int64_t ws_d0, int64_t ws_s0, int32_t dtype, int32_t store, void *stream) {
  const Arguments a{VIEW3(k), VIEW3(v), slots, slots_d0, slots_s0,
                    {VIEW4(k_cache), VIEW4(v_cache), VIEW3(k_scale), VIEW3(v_scale)},
                    workspace, ws_d0, ws_s0, dtype, store};
  const int status = check("cache_read", a, false);
  if (status != B200_OK) return status;
  if (!k_d0 || !k_d1) return B200_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (store == B200_F16 || store == B200_BF16)
    return dtype == B200_F16 ? by_lanes<kReadNative, __half, 1>(a, s) : by_lanes<kReadNative, __nv_bfloat16, 1>(a, s);
  return dtype == B200_F16 ? by_lanes<kRead, __half, 1>(a, s) : by_lanes<kRead, __nv_bfloat16, 1>(a, s);
}
