// Writing rows of keys and values into a paged cache and reading them back, in 16 or 8 bits.
//
// Both directions are bound by HBM: 2 bytes an element on the rows' side, 1 or 2 on the cache's and
// 4 for a row's scale.  A row of D columns belongs to D / 16 lanes of a warp (rounded up to a power
// of two), 16 columns a lane: two 128-bit vectors of rows against one of codes (two in 16 bits), the
// row's largest magnitude by a butterfly over those lanes.  One launch moves keys and values: a unit
// is the key row and the value row of one head of a token.
//
// Measured for 32768 tokens of 8 heads of 128 columns (bf16 rows, pages of 16 in any order; floors at the
// 6447 GB/s of a copy): 16 bits written in 41.8 us and read in 44 (41.7); int8 written in 38.5 us, read
// in 35.4 (31.6); e4m3 written in 34.1, read in 38.5 (31.6).  int8 is written at 82% of the copy's rate, held
// up by the exact quotients; reading writes two bytes for each that it reads.
#include "cache.cuh"

namespace b200 {
namespace {

using cache::Cache;
using heads::Eight;
using heads::View1;
using heads::View3;
using heads::View4;

using heads::kThreads;

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
  int tokens, heads, columns, page_size, store;
  int *status;
};

// Slot of a token, or -1 where there is none (padding; a slot behind the cache, which is reported).
__device__ __forceinline__ int64_t slot_of(const Extents &x, int token, bool first_lane) {
  const int64_t slot = x.slots[token * x.slots_step];
  if (slot < x.capacity) return slot < 0 ? -1 : slot;
  if (first_lane) heads::report_index(x.status, token);
  return -1;
}

// Bits of the largest magnitude, a NaN's if there is one.
__device__ __forceinline__ __half2 larger(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 larger(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <typename T> __device__ __forceinline__ uint32_t magnitude(const Eight<T> &a, const Eight<T> &b) {
  using Two16 = typename Pair<T>::type;
  const uint32_t words[8] = {a.raw[0].x, a.raw[0].y, a.raw[0].z, a.raw[0].w, b.raw[0].x, b.raw[0].y, b.raw[0].z, b.raw[0].w};
  Two16 most = __habs2(*reinterpret_cast<const Two16 *>(&words[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) most = larger(most, __habs2(*reinterpret_cast<const Two16 *>(&words[i])));
  const uint32_t both = *reinterpret_cast<const uint32_t *>(&most) & 0x7fff7fffu;
  return max(both & 0xffffu, both >> 16);
}

// Blocks of 256 on an SM.  Writing codes, 6 rather than 4 cost 40 registers instead of 48 and gain 4% (32768
// tokens of 8 heads of 128 columns); two heads a unit or a ring of copies in shared memory, with more in flight
// on fewer warps, lost 4 to 20%: a row's quotients, not its bytes, are what warps wait for.  Reading codes
// waits for slots, then for rows that they name: 8 blocks gain 12% over 4.
constexpr int kWriteBlocks = 6, kReadBlocks = 8, kNativeBlocks = 6;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, kWriteBlocks)
cache_write_codes_kernel(Rows rows, Pages pages, Extents x) {
  heads::await_stream();
  const int e = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / (uint32_t)x.heads), head = (int)(unit - (uint32_t)token * x.heads);
  const bool live = token < x.tokens && e * 16 < x.columns;
  Eight<T> a[2], b[2];   // key, value
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a[i].clear();
    b[i].clear();
    if (live) {
      const T *from = i == 0 ? static_cast<const T *>(rows.k) + token * rows.k_token + head * rows.k_head
                             : static_cast<const T *>(rows.v) + token * rows.v_token + head * rows.v_head;
      a[i].load(from + e * 16);
      b[i].load(from + e * 16 + 8);
    }
  }
  const int64_t slot = token < x.tokens ? slot_of(x, token, e == 0) : -1;
  uint32_t most[2] = {magnitude(a[0], b[0]), magnitude(a[1], b[1])};
#pragma unroll
  for (int lane = LANES / 2; lane > 0; lane >>= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) most[i] = max(most[i], __shfl_xor_sync(0xffffffffu, most[i], lane));
  if (!live || slot < 0) return;
  int64_t page;
  int offset;
  cache::locate(slot, x.page_size, page, offset);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t bits = (uint16_t)most[i];
    const uint32_t wide = __float_as_uint(Element<T>::widen(*reinterpret_cast<const T *>(&bits)));
    const float scale = x.store == cache::kInt8 ? cache::int8_scale(wide) : cache::e4m3_scale(wide);
    float values[16];
    a[i].widen(values);
    b[i].widen(values + 8);
    uint8_t *to = static_cast<uint8_t *>(i == 0 ? pages.k : pages.v) +
                  (i == 0 ? page * pages.k_page + head * pages.k_head + offset * pages.k_slot
                          : page * pages.v_page + head * pages.v_head + offset * pages.v_slot);
    *reinterpret_cast<uint4 *>(to + e * 16) = cache::encode(values, x.store, scale);
    if (e == 0)
      *(i == 0 ? pages.k_scale + page * pages.ks_page + head * pages.ks_head + offset * pages.ks_slot
               : pages.v_scale + page * pages.vs_page + head * pages.vs_head + offset * pages.vs_slot) = scale;
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, kReadBlocks)
cache_read_codes_kernel(Rows rows, Pages pages, Extents x) {
  heads::await_stream();
  const int e = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / (uint32_t)x.heads), head = (int)(unit - (uint32_t)token * x.heads);
  if (token >= x.tokens || e * 16 >= x.columns) return;
  const int64_t slot = slot_of(x, token, e == 0);
  uint4 codes[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};   // key, value
  float scale[2] = {0.0f, 0.0f};
  if (slot >= 0) {
    int64_t page;
    int offset;
    cache::locate(slot, x.page_size, page, offset);
    const uint8_t *k = static_cast<const uint8_t *>(pages.k) + page * pages.k_page + head * pages.k_head + offset * pages.k_slot;
    const uint8_t *v = static_cast<const uint8_t *>(pages.v) + page * pages.v_page + head * pages.v_head + offset * pages.v_slot;
    codes[0] = *reinterpret_cast<const uint4 *>(k + e * 16);
    codes[1] = *reinterpret_cast<const uint4 *>(v + e * 16);
    scale[0] = pages.k_scale[page * pages.ks_page + head * pages.ks_head + offset * pages.ks_slot];
    scale[1] = pages.v_scale[page * pages.vs_page + head * pages.vs_head + offset * pages.vs_slot];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float values[16];
    cache::decode(codes[i], x.store, scale[i], values);
    Eight<T> a, b;
    a.narrow(values);
    b.narrow(values + 8);
    T *to = i == 0 ? static_cast<T *>(rows.k) + token * rows.k_token + head * rows.k_head
                   : static_cast<T *>(rows.v) + token * rows.v_token + head * rows.v_head;
    a.store(to + e * 16);
    b.store(to + e * 16 + 8);
  }
}

// A 16-bit cache takes its rows and gives them back as they are.
template <typename T, int LANES, bool WRITE>
__global__ void __launch_bounds__(kThreads, kNativeBlocks)
cache_copy_kernel(Rows rows, Pages pages, Extents x) {
  heads::await_stream();
  const int e = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int token = (int)(unit / (uint32_t)x.heads), head = (int)(unit - (uint32_t)token * x.heads);
  if (token >= x.tokens || e * 16 >= x.columns) return;
  Eight<T> a[2], b[2];   // key, value
  T *k_row = static_cast<T *>(rows.k) + token * rows.k_token + head * rows.k_head + e * 16;
  T *v_row = static_cast<T *>(rows.v) + token * rows.v_token + head * rows.v_head + e * 16;
  if (WRITE) {           // the rows need not wait for the slot
    a[0].load(k_row);
    b[0].load(k_row + 8);
    a[1].load(v_row);
    b[1].load(v_row + 8);
  }
  const int64_t slot = slot_of(x, token, e == 0);
  if (slot < 0) {
    if (WRITE) return;
    a[0].clear();
    a[0].store(k_row);
    a[0].store(k_row + 8);
    a[0].store(v_row);
    a[0].store(v_row + 8);
    return;
  }
  int64_t page;
  int offset;
  cache::locate(slot, x.page_size, page, offset);
  T *k_held = static_cast<T *>(pages.k) + page * pages.k_page + head * pages.k_head + offset * pages.k_slot + e * 16;
  T *v_held = static_cast<T *>(pages.v) + page * pages.v_page + head * pages.v_head + offset * pages.v_slot + e * 16;
  if (!WRITE) {
    a[0].load(k_held);
    b[0].load(k_held + 8);
    a[1].load(v_held);
    b[1].load(v_held + 8);
  }
  a[0].store(WRITE ? k_held : k_row);
  b[0].store((WRITE ? k_held : k_row) + 8);
  a[1].store(WRITE ? v_held : v_row);
  b[1].store((WRITE ? v_held : v_row) + 8);
}

// --------------------------------------------------------------------- host
struct Arguments {
  View3 k, v;
  View1 slots;
  Cache cache;
  View1 workspace;
  int32_t dtype, store;
};

int check(const char *what, const Arguments &a, bool write) {
  if (a.dtype != B200_F16 && a.dtype != B200_BF16)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: rows are f16 or bf16", what);
  int status = cache::check(what, a.cache, a.dtype, a.store, 256);
  if (status != B200_OK) return status;
  const View4 &c = a.cache.k;
  if (!heads::sane(a.k) || !heads::sane(a.v) || !heads::sane(a.slots.d0, a.slots.s0))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (a.k.d0 != a.v.d0 || a.k.d0 != a.slots.d0) return fail(B200_ERR_INVALID_ARGUMENT, "%s: rows and slots differ in number", what);
  if (a.k.d1 != c.d1 || a.v.d1 != c.d1 || a.k.d2 != c.d3 || a.v.d2 != c.d3)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the rows' heads or columns are not the cache's", what);
  if (a.k.d0 >= (int64_t(1) << 31)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: 2^31 rows or more", what);
  if (!a.workspace.data || a.workspace.d0 < B200_WORKSPACE_WORDS || a.workspace.s0 != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the workspace needs %d contiguous int32 words", what, B200_WORKSPACE_WORDS);
  if (!heads::aligned4(a.workspace.data)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the workspace is 4-byte aligned", what);
  if (!a.k.d0 || !a.k.d1) return B200_OK;
  status = heads::check_units(what, a.k.d0, a.k.d1);
  if (status != B200_OK) return status;
  if (!a.k.data || !a.v.data || !a.slots.data) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(a.slots.data) & 7) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: slots are 8-byte aligned", what);
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
  using heads::footprint;
  const heads::Footprint space = footprint(a.workspace, 4), slots = footprint(a.slots, 8);
  const heads::Footprint rows[] = {footprint(a.k, 2), footprint(a.v, 2)}, codes[] = {footprint(a.cache.k, wide), footprint(a.cache.v, wide)};
  const heads::Footprint scales[] = {scaled ? footprint(a.cache.k_scale, 4) : heads::Footprint(),
                                     scaled ? footprint(a.cache.v_scale, 4) : heads::Footprint()};
  status = heads::check_written(what, &space, 1, &slots, 1);
  for (int i = 0; i < 2 && status == B200_OK; ++i) {
    const heads::Footprint around[] = {slots, space};
    status = heads::check_written(what, write ? &codes[i] : &rows[i], 1, around, 2);
    if (status == B200_OK && write) status = heads::check_written(what, &scales[i], 1, around, 2);
    if (status == B200_OK && write) status = heads::check_written(what, &scales[i], 1, codes, 2);
    if (status == B200_OK) status = heads::check_written(what, &space, 1, write ? rows : codes, 2);
    if (status == B200_OK && !write) status = heads::check_written(what, &space, 1, scales, 2);
  }
  return status;
}

void pack(const Arguments &a, Rows &rows, Pages &pages, Extents &x) {
  rows = {const_cast<void *>(a.k.data), const_cast<void *>(a.v.data), a.k.s0, a.k.s1, a.v.s0, a.v.s1};
  const Cache &c = a.cache;
  pages = {const_cast<void *>(c.k.data), const_cast<void *>(c.v.data), c.k.s0, c.k.s1, c.k.s2, c.v.s0, c.v.s1, c.v.s2,
           static_cast<float *>(const_cast<void *>(c.k_scale.data)), static_cast<float *>(const_cast<void *>(c.v_scale.data)),
           c.k_scale.s0, c.k_scale.s1, c.k_scale.s2, c.v_scale.s0, c.v_scale.s1, c.v_scale.s2};
  x = {};
  x.slots = static_cast<const int64_t *>(a.slots.data);
  x.slots_step = a.slots.s0;
  x.capacity = c.k.d0 * c.k.d2;
  x.tokens = (int)a.k.d0;
  x.heads = (int)c.k.d1;
  x.columns = (int)c.k.d3;
  x.page_size = (int)c.k.d2;
  x.store = a.store == B200_I8 ? cache::kInt8 : a.store == B200_E4M3 ? cache::kE4m3 : cache::kNative;
  x.status = static_cast<int *>(const_cast<void *>(a.workspace.data));
}

template <typename T, int LANES> int launch(const Arguments &a, bool write, cudaStream_t stream) {
  Rows rows;
  Pages pages;
  Extents x;
  pack(a, rows, pages, x);
  const int64_t units = (int64_t)x.tokens * x.heads, per_block = kThreads / LANES;
  const unsigned blocks = (unsigned)((units + per_block - 1) / per_block);
  const auto kernel = x.store == cache::kNative ? (write ? cache_copy_kernel<T, LANES, true> : cache_copy_kernel<T, LANES, false>)
                      : write                   ? cache_write_codes_kernel<T, LANES>
                                                : cache_read_codes_kernel<T, LANES>;
  B200_CUDA_TRY(heads::launch_early(kernel, blocks, kThreads, 0, stream, rows, pages, x));
  return B200_OK;
}

template <typename T> int by_lanes(const Arguments &a, bool write, cudaStream_t stream) {
  switch (heads::row_lanes(a.cache.k.d3)) {
  case 1: return launch<T, 1>(a, write, stream);
  case 2: return launch<T, 2>(a, write, stream);
  case 4: return launch<T, 4>(a, write, stream);
  case 8: return launch<T, 8>(a, write, stream);
  default: return launch<T, 16>(a, write, stream);
  }
}

int run(const char *what, const Arguments &a, bool write, void *stream) {
  const int status = check(what, a, write);
  if (status != B200_OK || !a.k.d0 || !a.k.d1) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a.dtype == B200_F16 ? by_lanes<__half>(a, write, s) : by_lanes<__nv_bfloat16>(a, write, s);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_cache_write(const int64_t *slots, int64_t count, int32_t dtype, int32_t store, void *stream) {
  heads::Slots from(slots, count);
  Arguments a{};
  a.k = from.view3();
  a.v = from.view3();
  a.slots = from.view1();
  a.cache.k = from.view4();
  a.cache.v = from.view4();
  a.cache.k_scale = from.view3();
  a.cache.v_scale = from.view3();
  a.workspace = from.view1();
  if (!from.exact()) return fail(B200_ERR_INVALID_ARGUMENT, "cache_write: %lld slots do not describe its views", (long long)count);
  a.dtype = dtype;
  a.store = store;
  return run("cache_write", a, true, stream);
}

extern "C" int b200_cache_read(const int64_t *slots, int64_t count, int32_t dtype, int32_t store, void *stream) {
  heads::Slots from(slots, count);
  Arguments a{};
  a.cache.k = from.view4();
  a.cache.v = from.view4();
  a.slots = from.view1();
  a.cache.k_scale = from.view3();
  a.cache.v_scale = from.view3();
  a.k = from.view3();
  a.v = from.view3();
  a.workspace = from.view1();
  if (!from.exact()) return fail(B200_ERR_INVALID_ARGUMENT, "cache_read: %lld slots do not describe its views", (long long)count);
  a.dtype = dtype;
  a.store = store;
  return run("cache_read", a, false, stream);
}
