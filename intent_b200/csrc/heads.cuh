// Rows of attention heads: views, 16-column pieces of a row held by one lane, argument checks.
// Shared by the per-head norm and rotation, the paged cache and the attention over it.
#pragma once

#include <math.h>

#include "common.cuh"

namespace b200 {
namespace heads {

// ---- host: views as the ABI passes them -----------------------------------
struct View3 {
  const void *data;
  int64_t d0, d1, d2, s0, s1, s2;
};
struct View4 {
  const void *data;
  int64_t d0, d1, d2, d3, s0, s1, s2, s3;
};

struct View2 {
  const void *data;
  int64_t d0, d1, s0, s1;
};
struct View1 {
  const void *data;
  int64_t d0, s0;
};

// Takes views off an array of slots: pointer, extents, strides of each, as the ABI orders them.
class Slots {
 public:
  Slots(const int64_t *words, int64_t count) : words_(words), count_(words ? count : 0) {}
  View1 view1() { return {pointer(), next(), next()}; }
  View2 view2() { return {pointer(), next(), next(), next(), next()}; }
  View3 view3() { return {pointer(), next(), next(), next(), next(), next(), next()}; }
  View4 view4() { return {pointer(), next(), next(), next(), next(), next(), next(), next(), next()}; }
  bool exact() const { return taken_ == count_; }   // neither more nor fewer than there are

 private:
  int64_t next() { return taken_++ < count_ ? words_[taken_ - 1] : 0; }
  const void *pointer() { return reinterpret_cast<const void *>(next()); }
  const int64_t *words_;
  int64_t count_, taken_ = 0;
};

inline int element_size(int dtype) { return dtype == B200_F32 ? 4 : dtype == B200_F16 || dtype == B200_BF16 ? 2 : 1; }

// Strides times extents, added up over four axes and in bytes, stay below 2^61, whatever the caller passes.
inline bool sane(int64_t extent, int64_t stride) {
  return extent >= 0 && extent < (int64_t(1) << 40) && stride > -(int64_t(1) << 40) && stride < (int64_t(1) << 40) &&
         (extent <= 1 || llabs(stride) <= (int64_t(1) << 57) / extent);
}
inline bool sane(const View3 &v) { return sane(v.d0, v.s0) && sane(v.d1, v.s1) && sane(v.d2, v.s2); }
inline bool sane(const View4 &v) { return sane(v.d0, v.s0) && sane(v.d1, v.s1) && sane(v.d2, v.s2) && sane(v.d3, v.s3); }

// Words that kernels load and store one by one: a misaligned one would fault.
inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Rows move as 128-bit vectors: unit innermost stride, 16-byte aligned base and outer strides.
inline bool vector_rows(const View3 &v, int size) {
  const int64_t step = 16 / size;
  return v.s2 == 1 && aligned16(v.data) && (v.d0 <= 1 || v.s0 % step == 0) && (v.d1 <= 1 || v.s1 % step == 0);
}
inline bool vector_rows(const View4 &v, int size) {
  const int64_t step = 16 / size;
  return v.s3 == 1 && aligned16(v.data) && (v.d0 <= 1 || v.s0 % step == 0) && (v.d1 <= 1 || v.s1 % step == 0) &&
         (v.d2 <= 1 || v.s2 % step == 0);
}

struct Span {
  uintptr_t begin, end;
};
inline Span span(const void *data, int size, int count, const int64_t *extents, const int64_t *strides) {
  int64_t low = 0, high = 0;
  for (int i = 0; i < count; ++i) {
    if (extents[i] == 0) return {0, 0};
    const int64_t reach = (extents[i] - 1) * strides[i];
    (reach < 0 ? low : high) += reach;
  }
  const uintptr_t base = reinterpret_cast<uintptr_t>(data);
  return {base + low * size, base + (high + 1) * size};
}
inline Span span(const View3 &v, int size) {
  const int64_t extents[] = {v.d0, v.d1, v.d2}, strides[] = {v.s0, v.s1, v.s2};
  return span(v.data, size, 3, extents, strides);
}
inline Span span(const View4 &v, int size) {
  const int64_t extents[] = {v.d0, v.d1, v.d2, v.d3}, strides[] = {v.s0, v.s1, v.s2, v.s3};
  return span(v.data, size, 4, extents, strides);
}
inline bool overlap(const Span &a, const Span &b) { return a.begin < b.end && b.begin < a.end; }

// Whether two elements of a view that is written share an address: a sufficient test that every
// layout made by permuting and slicing a dense tensor passes.  Axes in the order of their strides;
// each must step over all that the smaller ones reach.
inline bool distinct(int count, const int64_t *extents, const int64_t *strides) {
  int order[5];
  for (int i = 0; i < count; ++i) {
    if (extents[i] == 0) return true;
    order[i] = i;
  }
  for (int i = 1; i < count; ++i)
    for (int j = i; j > 0 && llabs(strides[order[j]]) < llabs(strides[order[j - 1]]); --j) {
      const int other = order[j];
      order[j] = order[j - 1];
      order[j - 1] = other;
    }
  int64_t reach = 0;
  for (int i = 0; i < count; ++i) {
    const int axis = order[i];
    if (extents[axis] == 1) continue;
    if (llabs(strides[axis]) <= reach) return false;
    reach += (extents[axis] - 1) * llabs(strides[axis]);
  }
  return true;
}
inline bool distinct(const View3 &v) {
  const int64_t extents[] = {v.d0, v.d1, v.d2}, strides[] = {v.s0, v.s1, v.s2};
  return distinct(3, extents, strides);
}
inline bool distinct(const View4 &v) {
  const int64_t extents[] = {v.d0, v.d1, v.d2, v.d3}, strides[] = {v.s0, v.s1, v.s2, v.s3};
  return distinct(4, extents, strides);
}

// Whether two views that are written share no element, by a sufficient test: they lie apart, or they
// have one shape and one layout and interleave (keys and values of one allocation).
inline bool apart(const View4 &a, const View4 &b, int size) {
  if (!overlap(span(a, size), span(b, size))) return true;
  const int64_t extents[] = {a.d0, a.d1, a.d2, a.d3, 2};
  const int64_t strides[] = {a.s0, a.s1, a.s2, a.s3, ((const char *)b.data - (const char *)a.data) / size};
  if (a.d0 != b.d0 || a.d1 != b.d1 || a.d2 != b.d2 || a.d3 != b.d3 || (a.d0 > 1 && a.s0 != b.s0) || (a.d1 > 1 && a.s1 != b.s1) ||
      (a.d2 > 1 && a.s2 != b.s2) || (a.d3 > 1 && a.s3 != b.s3))
    return false;
  return distinct(5, extents, strides);
}
inline bool apart(const View3 &a, const View3 &b, int size) {
  return apart(View4{a.data, a.d0, a.d1, a.d2, 1, a.s0, a.s1, a.s2, 1}, View4{b.data, b.d0, b.d1, b.d2, 1, b.s0, b.s1, b.s2, 1}, size);
}

// Where a view's elements lie: its lowest address, and the axes that move, the longest steps first (bytes).
struct Footprint {
  int64_t base = 0, element = 0;   // element 0: nothing
  int axes = 0;
  int64_t extents[4], steps[4];
  Footprint() = default;
  Footprint(const void *data, int size, int count, const int64_t *counts, const int64_t *strides)
      : base((int64_t)reinterpret_cast<uintptr_t>(data)), element(size) {
    for (int i = 0; i < count; ++i) {
      if (counts[i] == 0) element = 0;
      if (counts[i] <= 1 || strides[i] == 0) continue;
      if (strides[i] < 0) base += (counts[i] - 1) * strides[i] * size;
      const int64_t step = llabs(strides[i]) * size;
      int at = axes++;
      for (; at > 0 && steps[at - 1] < step; --at) {
        extents[at] = extents[at - 1];
        steps[at] = steps[at - 1];
      }
      extents[at] = counts[i];
      steps[at] = step;
    }
  }
  int64_t length(int axis) const {   // of what the axes from `axis` on reach
    int64_t bytes = element;
    for (int i = axis; i < axes; ++i) bytes += (extents[i] - 1) * steps[i];
    return bytes;
  }
};
inline Footprint footprint(const View1 &v, int size) { return Footprint(v.data, size, 1, &v.d0, &v.s0); }
inline Footprint footprint(const View2 &v, int size) {
  const int64_t extents[] = {v.d0, v.d1}, strides[] = {v.s0, v.s1};
  return Footprint(v.data, size, 2, extents, strides);
}
inline Footprint footprint(const View3 &v, int size) {
  const int64_t extents[] = {v.d0, v.d1, v.d2}, strides[] = {v.s0, v.s1, v.s2};
  return Footprint(v.data, size, 3, extents, strides);
}
inline Footprint footprint(const View4 &v, int size) {
  const int64_t extents[] = {v.d0, v.d1, v.d2, v.d3}, strides[] = {v.s0, v.s1, v.s2, v.s3};
  return Footprint(v.data, size, 4, extents, strides);
}

// Whether two views share no byte, by a sufficient test: one ends before the other begins, or their longest steps are
// alike and what lies inside a step is apart, seen from this step and from the next (a cache's pages with their scales
// behind the codes).  b's part begins `gap` bytes behind a's.
inline bool disjoint(const Footprint &a, const Footprint &b, int axis, int64_t gap) {
  if (!a.element || !b.element || gap >= a.length(axis) || gap + b.length(axis) <= 0) return true;
  if (axis >= a.axes || axis >= b.axes || a.steps[axis] != b.steps[axis]) return false;
  const int64_t step = a.steps[axis], inside = ((gap % step) + step) % step;
  if (a.length(axis + 1) > step || b.length(axis + 1) > step) return false;
  return disjoint(a, b, axis + 1, inside) && disjoint(a, b, axis + 1, inside - step);
}
inline bool disjoint(const Footprint &a, const Footprint &b) { return disjoint(a, b, 0, b.base - a.base); }

// What a call writes meets neither what it reads nor anything else that it writes.
inline int check_written(const char *what, const Footprint *written, int count, const Footprint *read, int reads) {
  for (int i = 0; i < count; ++i) {
    for (int j = 0; j < reads; ++j)
      if (!disjoint(written[i], read[j])) return fail(B200_ERR_INVALID_ARGUMENT, "%s: an output overlaps an operand", what);
    for (int j = 0; j < i; ++j)
      if (!disjoint(written[i], written[j])) return fail(B200_ERR_INVALID_ARGUMENT, "%s: two outputs (or scratch) overlap", what);
  }
  return B200_OK;
}

// Lanes that share a row when each holds 16 of its columns: a power of two, so that a warp holds
// whole rows and the sum over a row is a butterfly of shuffles.
inline int row_lanes(int64_t columns) {
  int lanes = 1;
  while (lanes * 16 < columns) lanes *= 2;
  return lanes;
}

// Threads of a block of the kernels that move rows.
constexpr int kThreads = 256;

inline int check_units(const char *what, int64_t tokens, int64_t slices) {
  if (tokens * slices >= (int64_t(1) << 32) - (1 << 21))   // counted in 32 bits: a 64-bit division costs as much as a row's arithmetic
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: 2^32 rows or more in one call", what);
  return B200_OK;
}

// Launches a kernel whose blocks may be placed while the stream's kernel before it ends.  Every block of
// such a kernel begins with await_stream() and touches no memory before that, so the stream's order holds; it
// saves the 2 us that a kernel of a few microseconds otherwise waits for its predecessor's last block.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_early(void (*kernel)(Parameters...), dim3 blocks, unsigned threads, size_t smem, cudaStream_t stream,
                         Arguments... arguments) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = blocks;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

// ---- device ------------------------------------------------------------------
// Waits until what the stream held before this kernel is done and seen; then lets the next kernel's blocks in.
__device__ __forceinline__ void await_stream() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Word kBadIndex of the workspace becomes 1 and the next one the position of a bad index (b200_workspace_status
// reports it); the first one found stays.  Words 0 and 1 belong to waits that give up, which a bad index must not hide.
__device__ __forceinline__ void report_index(int *status, int position) {
  if (atomicCAS(status + kBadIndex, 0, 1) == 0) status[kBadIndex + 1] = position;
}

// Two f32 at a time (one instruction each on this part).
struct Two {
  float a, b;
};
__device__ __forceinline__ uint64_t bits(Two v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.a), "f"(v.b));
  return r;
}
__device__ __forceinline__ Two two(uint64_t v) {
  Two r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.a), "=f"(r.b) : "l"(v));
  return r;
}
__device__ __forceinline__ Two mul(Two x, Two y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(x)), "l"(bits(y)));
  return two(r);
}
__device__ __forceinline__ Two fma(Two x, Two y, Two z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(x)), "l"(bits(y)), "l"(bits(z)));
  return two(r);
}
__device__ __forceinline__ Two swap(Two x) { return {x.b, x.a}; }

// Eight consecutive columns, as raw 128-bit vectors and as f32.
template <typename T> struct Eight {
  static constexpr int kVectors = 8 * sizeof(T) / 16;
  uint4 raw[kVectors];
  __device__ __forceinline__ void load(const T *pointer) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) raw[i] = reinterpret_cast<const uint4 *>(pointer)[i];
  }
  __device__ __forceinline__ void store(T *pointer) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) reinterpret_cast<uint4 *>(pointer)[i] = raw[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void widen(float *out) const {
    const T *lanes = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = Element<T>::widen(lanes[i]);
  }
  __device__ __forceinline__ void narrow(const float *in) {
    T *lanes = reinterpret_cast<T *>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) lanes[i] = Element<T>::narrow(in[i]);
  }
};

template <int LANES> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int offset = LANES / 2; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

}  // namespace heads
}  // namespace b200
