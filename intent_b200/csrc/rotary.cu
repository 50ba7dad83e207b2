// RMS norm of every query and key head and the rotation by its token's position, one pass.
//
//     r = 1 / sqrt(mean(x^2) + eps)      z = x r w      y = R(position) z
//
// R turns the pairs (z_a, z_b) of the first 2 * half columns, (i, i + half) or (2i, 2i + 1), by the
// angle whose cosine and sine the caller's f32 tables hold at [position, i]; later columns pass.
// R is orthogonal, so with g = R^T dy and u = g w the backward pass is
//
//     dw = sum over rows of g x r        dx = r (u - x r mean(u x r))
//
// Both are bound by HBM: a row is read once, kept in registers as f32, and written once.  A row of
// D columns belongs to D / 16 lanes of a warp (rounded up to a power of two), each of which holds
// 16 columns as two 128-bit vectors (16-bit types) chosen so that BOTH ends of its pairs are its own:
// the rotation needs no exchange, the mean is a butterfly over those lanes.  The 8 cosines and 8
// sines that a lane needs are loaded once for all the heads that it takes of a token.
//
// Rows arrive by cp.async in places of shared memory that are each thread's own, several rows ahead: what is
// in flight takes no registers, and 16 warps of an SM keep 64 KB and more on their way.  Arithmetic is on
// pairs of f32.  Measured for 16384 tokens of 32 and 8 heads of 128 columns in bf16: 58 us forward, 5.8 TB/s
// (337 MB; 52 us at the 6447 GB/s of a copy), 86 us backward, 5.8 TB/s (504 MB; 78 us).  Without the
// ring and the pairs, one row a thread at a time: 77 and 138 us.
#include "heads.cuh"

namespace b200 {
namespace {

using heads::Eight;
using heads::fma;
using heads::mul;
using heads::swap;
using heads::Two;
using heads::View1;
using heads::View2;
using heads::View3;

using heads::kThreads;

constexpr int kBlocksPerSm = 2;

struct Operand {        // one of q, k (and, for the backward pass, its gradients)
  const void *x;
  const void *grad;     // backward only
  const void *weight;
  void *out;
  int64_t x_token, x_head, grad_token, grad_head, out_token, out_head;
  int heads;
  uint32_t slices;      // units per token: ceil(heads / rows of a unit)
};

struct Rotation {
  const float *cosine, *sine;
  int64_t cosine_row, sine_row;
  int table_rows, half, columns;
  int interleaved;
  const int *positions;
  int64_t positions_step;
  int tokens;
  float inverse_columns, epsilon;
  int *status;
};

// The two pieces of 8 columns that lane `e` of a row holds.  Inside the rotated columns the pieces
// are 8 pairs' first and second members (half split), or 16 neighbouring columns (interleaved and
// what passes unrotated).
__device__ __forceinline__ void pieces(const Rotation &r, int e, int &first, int &second) {
  const bool split = !r.interleaved && e * 8 < r.half;
  first = split ? 8 * e : 16 * e;
  second = split ? r.half + 8 * e : 16 * e + 8;
}

// 16 columns of a row, neighbours in pairs: own[0..4) is the first piece and own[4..8) the second.
struct Row {
  Two own[8];
  template <typename T> __device__ __forceinline__ void widen(const Eight<T> &a, const Eight<T> &b) {
    float x[16];
    a.widen(x);
    b.widen(x + 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = {x[2 * i], x[2 * i + 1]};
  }
  template <typename T> __device__ __forceinline__ void narrow(Eight<T> &a, Eight<T> &b) const {
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) { x[2 * i] = own[i].a; x[2 * i + 1] = own[i].b; }
    a.narrow(x);
    b.narrow(x + 8);
  }
  __device__ __forceinline__ float dot(const Row &other) const {
    Two sum = mul(own[0], other.own[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) sum = fma(own[i], other.own[i], sum);
    return sum.a + sum.b;
  }
};

// A turn as y = x * straight + partner(x) * crossed, where a column's partner is the other member of
// its pair.  Lanes whose columns pass never look at partners: an infinity there times 0 would be NaN.
__device__ __forceinline__ Row turned_row(const Row &x, const Row &straight, const Row &crossed, bool turned, bool interleaved) {
  Row y;
  if (!turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y.own[i] = mul(x.own[i], straight.own[i]);
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y.own[i] = fma(x.own[i], straight.own[i], mul(swap(x.own[i]), crossed.own[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y.own[i] = fma(x.own[i], straight.own[i], mul(x.own[(i + 4) & 7], crossed.own[i]));
  }
  return y;
}

// straight and crossed of R (BACK: of its transpose) for lane `e` at a position.
template <bool BACK>
__device__ __forceinline__ void angles(const Rotation &r, int e, int position, Row &straight, Row &crossed) {
  const float4 *c4 = reinterpret_cast<const float4 *>(r.cosine + position * r.cosine_row + 8 * e);
  const float4 *s4 = reinterpret_cast<const float4 *>(r.sine + position * r.sine_row + 8 * e);
  const float4 c0 = __ldg(c4), c1 = __ldg(c4 + 1), s0 = __ldg(s4), s1 = __ldg(s4 + 1);
  const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
  if (r.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      straight.own[i] = {c[i], c[i]};
      crossed.own[i] = BACK ? Two{s[i], -s[i]} : Two{-s[i], s[i]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      straight.own[i] = straight.own[i + 4] = {c[2 * i], c[2 * i + 1]};
      const Two positive = {s[2 * i], s[2 * i + 1]}, negative = {-s[2 * i], -s[2 * i + 1]};
      crossed.own[i] = BACK ? positive : negative;
      crossed.own[i + 4] = BACK ? negative : positive;
    }
  }
}

// Position of a token, or -1 where its rows are zeros (padding; a place behind the tables, which is reported).
__device__ __forceinline__ int place(const Rotation &r, int token, bool first_lane) {
  const int position = r.positions[token * r.positions_step];
  if (position < r.table_rows) return position < 0 ? -1 : position;
  if (first_lane) heads::report_index(r.status, token);
  return -1;
}

// A group's place in the grid of units: a division at the start, additions from then on.
struct Cursor {
  uint32_t base, token, slice;      // base: the block's first unit of the round
  __device__ __forceinline__ Cursor(uint32_t first, uint32_t group, uint32_t slices)
      : base(first), token((first + group) / slices), slice((first + group) % slices) {}
  __device__ __forceinline__ void advance(uint32_t step, uint32_t step_token, uint32_t step_slice, uint32_t slices) {
    base += step;
    token += step_token;
    slice += step_slice;
    if (slice >= slices) {
      slice -= slices;
      ++token;
    }
  }
};

// Rows on their way to a thread: each copies its own pieces of the rows it will take into its own
// places of shared memory (16 bytes a thread, neighbours side by side) STAGES - 1 rows ahead, so that
// what is in flight does not take registers and nobody waits for anybody else.
template <int VECTORS, int STAGES> struct Ring {
  static constexpr int kBytes = VECTORS * STAGES * kThreads * 16;
  uint4 *mine;
  uint32_t address;
  __device__ __forceinline__ explicit Ring(unsigned char *smem) {
    mine = reinterpret_cast<uint4 *>(smem) + threadIdx.x;
    address = (uint32_t)__cvta_generic_to_shared(mine);
  }
  template <typename T> __device__ __forceinline__ void copy(int stage, int vector, const T *from, bool live) const {
#pragma unroll
    for (int i = 0; i < Eight<T>::kVectors; ++i)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       address + ((stage * VECTORS + vector * Eight<T>::kVectors + i) * kThreads) * 16),
                   "l"(reinterpret_cast<const uint4 *>(from) + i), "r"(live ? 16 : 0) : "memory");
  }
  template <typename T> __device__ __forceinline__ Eight<T> take(int stage, int vector) const {
    Eight<T> v;
#pragma unroll
    for (int i = 0; i < Eight<T>::kVectors; ++i)
      v.raw[i] = mine[(stage * VECTORS + vector * Eight<T>::kVectors + i) * kThreads];
    return v;
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
};

// ------------------------------------------------------------------ forward
// A unit is `unit_rows` heads of one token, all of q or all of k; they share one load of the cosines,
// sines and weights, whose products (32 registers) are all that a row's turn needs.
template <typename T> constexpr int kForwardStages = sizeof(T) == 2 ? 6 : 4;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
head_norm_rotary_kernel(Operand q, Operand k, Rotation r, int unit_rows, uint32_t units) {
  constexpr int kGroups = kThreads / LANES, kStages = kForwardStages<T>;
  using Copies = Ring<2 * Eight<T>::kVectors, kStages>;
  extern __shared__ __align__(16) unsigned char dynamic_smem[];
  const Copies ring(dynamic_smem);
  heads::await_stream();
  const int e = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const uint32_t slices = q.slices + k.slices, step = gridDim.x * kGroups;
  const bool inside = e * 16 < r.columns, interleaved = r.interleaved;
  int first, second;
  pieces(r, e, first, second);

  // every group of the block runs the same number of rounds: the shuffles below are whole-warp
  const uint32_t step_token = step / slices, step_slice = step % slices;
  Cursor load(blockIdx.x * kGroups, group, slices);
  Cursor use = load;
  int load_row = 0, load_rows = 0;
  const T *source = nullptr;
  int64_t source_head = 0;
  auto produce = [&](int stage) {
    if (load.base < units) {
      if (load_row == 0) {
        const bool is_key = load.slice >= q.slices;
        const Operand &o = is_key ? k : q;
        const int head0 = (int)(is_key ? load.slice - q.slices : load.slice) * unit_rows;
        load_rows = load.base + group < units && inside ? min(unit_rows, o.heads - head0) : 0;
        source_head = o.x_head;
        source = static_cast<const T *>(o.x) + (load_rows ? load.token * o.x_token + head0 * o.x_head : 0);
      }
      const T *from = load_row < load_rows ? source + load_row * source_head : source;
      ring.template copy<T>(stage, 0, from + first, load_row < load_rows);
      ring.template copy<T>(stage, 1, from + second, load_row < load_rows);
      if (++load_row == unit_rows) {
        load_row = 0;
        load.advance(step, step_token, step_slice, slices);
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) produce(i);
  int stage = 0;
  for (; use.base < units; use.advance(step, step_token, step_slice, slices)) {
    const uint32_t unit = use.base + group, token = use.token;
    const bool is_key = use.slice >= q.slices, live = unit < units && inside;
    const Operand &o = is_key ? k : q;
    const int head0 = (int)(is_key ? use.slice - q.slices : use.slice) * unit_rows, rows = live ? min(unit_rows, o.heads - head0) : 0;
    const int position = unit < units ? place(r, token, e == 0) : -1;
    const bool turned = live && e * 8 < r.half && position >= 0;
    Row straight, crossed, w;
    if (live) {
      const T *weight = static_cast<const T *>(o.weight);
      Eight<T> w0, w1;
      w0.load(weight + first);
      w1.load(weight + second);
      w.widen(w0, w1);
    }
    if (turned) {
      angles<false>(r, e, position, straight, crossed);
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // the partner's weight goes with the partner
        crossed.own[i] = mul(crossed.own[i], interleaved ? swap(w.own[i]) : w.own[(i + 4) & 7]);
        straight.own[i] = mul(straight.own[i], w.own[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) straight.own[i] = w.own[i];
    }
    T *target = static_cast<T *>(o.out) + (live ? token * o.out_token + head0 * o.out_head : 0);
#pragma unroll 1
    for (int row = 0; row < unit_rows; ++row) {
      produce(stage == 0 ? kStages - 1 : stage - 1);
      ring.wait();
      Row x;
      x.widen(ring.template take<T>(stage, 0), ring.template take<T>(stage, 1));
      stage = stage == kStages - 1 ? 0 : stage + 1;
      const float squares = heads::row_sum<LANES>(x.dot(x));
      const float rstd = rsqrtf(squares * r.inverse_columns + r.epsilon);
#pragma unroll
      for (int i = 0; i < 8; ++i) x.own[i] = mul(x.own[i], Two{rstd, rstd});
      if (row < rows) {
        Eight<T> a, b;
        if (position < 0) {
          a.clear();
          b.clear();
        } else {
          turned_row(x, straight, crossed, turned, interleaved).narrow(a, b);
        }
        a.store(target + row * o.out_head + first);
        b.store(target + row * o.out_head + second);
      }
    }
  }
}

// ----------------------------------------------------------------- backward
// The blocks of [0, q_blocks) take q's units, the others k's, so that a lane keeps the sums of one
// weight only: 16 columns in f32, over all the rows it meets.  A block adds its lanes' sums in a
// fixed order and writes one row of `partial`; the second kernel adds those rows, again in a fixed
// order, so that dw does not vary from run to run.
template <typename T> constexpr int kBackwardStages = sizeof(T) == 2 ? 5 : 3;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
head_norm_rotary_backward_kernel(Operand q, Operand k, Rotation r, int unit_rows, int q_blocks, float *__restrict__ partial) {
  constexpr int kGroups = kThreads / LANES, kStages = kBackwardStages<T>;
  using Copies = Ring<4 * Eight<T>::kVectors, kStages>;
  static_assert(Copies::kBytes >= kGroups * (LANES * 16 + 1) * 4, "the ring holds the block's sums in the end");
  extern __shared__ __align__(16) unsigned char dynamic_smem[];
  const Copies ring(dynamic_smem);
  heads::await_stream();
  const int e = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool is_key = (int)blockIdx.x >= q_blocks, interleaved = r.interleaved;
  const Operand o = is_key ? k : q;
  const uint32_t block = is_key ? blockIdx.x - q_blocks : blockIdx.x;
  const uint32_t step = (is_key ? gridDim.x - q_blocks : q_blocks) * kGroups, units = r.tokens * o.slices;
  const bool inside = e * 16 < r.columns;
  int first, second;
  pieces(r, e, first, second);
  Row w, dw;
#pragma unroll
  for (int i = 0; i < 8; ++i) w.own[i] = dw.own[i] = {0.0f, 0.0f};
  if (inside) {
    const T *weight = static_cast<const T *>(o.weight);
    Eight<T> w0, w1;
    w0.load(weight + first);
    w1.load(weight + second);
    w.widen(w0, w1);
  }
  const uint32_t step_token = step / o.slices, step_slice = step % o.slices;
  Cursor load(block * kGroups, group, o.slices);
  Cursor use = load;
  int load_row = 0, load_rows = 0;
  const T *x_source = nullptr, *grad_source = nullptr;
  auto produce = [&](int stage) {
    if (load.base < units) {
      if (load_row == 0) {
        const int head0 = (int)load.slice * unit_rows;
        load_rows = load.base + group < units && inside ? min(unit_rows, o.heads - head0) : 0;
        x_source = static_cast<const T *>(o.x) + (load_rows ? load.token * o.x_token + head0 * o.x_head : 0);
        grad_source = static_cast<const T *>(o.grad) + (load_rows ? load.token * o.grad_token + head0 * o.grad_head : 0);
      }
      const bool live = load_row < load_rows;
      const T *x = live ? x_source + load_row * o.x_head : x_source, *g = live ? grad_source + load_row * o.grad_head : grad_source;
      ring.template copy<T>(stage, 0, x + first, live);
      ring.template copy<T>(stage, 1, x + second, live);
      ring.template copy<T>(stage, 2, g + first, live);
      ring.template copy<T>(stage, 3, g + second, live);
      if (++load_row == unit_rows) {
        load_row = 0;
        load.advance(step, step_token, step_slice, o.slices);
      }
    }
    ring.commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) produce(i);
  int stage = 0;
  // every group of the block runs the same number of rounds: the shuffles below are whole-warp
  for (; use.base < units; use.advance(step, step_token, step_slice, o.slices)) {
    const uint32_t unit = use.base + group, token = use.token;
    const int head0 = (int)use.slice * unit_rows;
    const int rows = unit < units && inside ? min(unit_rows, o.heads - head0) : 0;
    const int position = unit < units ? place(r, token, e == 0) : -1;
    const bool turned = inside && e * 8 < r.half && position >= 0;
    Row straight, crossed;
    if (turned) {
      angles<true>(r, e, position, straight, crossed);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) straight.own[i] = {1.0f, 1.0f};
    }
    T *target = static_cast<T *>(o.out) + (rows ? token * o.out_token + head0 * o.out_head : 0);
#pragma unroll 1
    for (int row = 0; row < unit_rows; ++row) {
      produce(stage == 0 ? kStages - 1 : stage - 1);
      ring.wait();
      Row x, g;
      x.widen(ring.template take<T>(stage, 0), ring.template take<T>(stage, 1));
      g.widen(ring.template take<T>(stage, 2), ring.template take<T>(stage, 3));
      stage = stage == kStages - 1 ? 0 : stage + 1;
      if (position < 0) {   // padding may hold anything, and adds nothing
#pragma unroll
        for (int i = 0; i < 8; ++i) x.own[i] = g.own[i] = {0.0f, 0.0f};
      }
      const float squares = heads::row_sum<LANES>(x.dot(x));
      // 0 where nothing counts: with epsilon 0 a row of zeros has no finite one
      const float rstd = row < rows && position >= 0 ? rsqrtf(squares * r.inverse_columns + r.epsilon) : 0.0f;
      g = turned_row(g, straight, crossed, turned, interleaved);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x.own[i] = mul(x.own[i], Two{rstd, rstd});
        dw.own[i] = fma(g.own[i], x.own[i], dw.own[i]);
        g.own[i] = mul(g.own[i], w.own[i]);
      }
      const float projection = -heads::row_sum<LANES>(g.dot(x)) * r.inverse_columns;
      if (row < rows) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          g.own[i] = mul(fma(x.own[i], Two{projection, projection}, g.own[i]), Two{rstd, rstd});
        Eight<T> a, b;
        g.narrow(a, b);
        if (position < 0) {   // 0 times a weight may be NaN
          a.clear();
          b.clear();
        }
        a.store(target + row * o.out_head + first);
        b.store(target + row * o.out_head + second);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float(*sums)[LANES * 16 + 1] = reinterpret_cast<float(*)[LANES * 16 + 1]>(dynamic_smem);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sums[group][2 * i * LANES + e] = dw.own[i].a;
    sums[group][(2 * i + 1) * LANES + e] = dw.own[i].b;
  }
  __syncthreads();
  for (int slot = threadIdx.x; slot < LANES * 16; slot += kThreads) {
    const int owner = slot % LANES, i = slot / LANES;
    if (owner * 16 >= r.columns) continue;
    float total = 0.0f;
#pragma unroll 8
    for (int g = 0; g < kGroups; ++g) total += sums[g][slot];
    int a, b;
    pieces(r, owner, a, b);
    partial[(int64_t)blockIdx.x * r.columns + (i < 8 ? a + i : b + i - 8)] = total;
  }
}

// 32 columns x 32 lanes of rows: even blocks add q's rows of `partial`, odd ones k's.
__global__ void __launch_bounds__(1024)
head_norm_rotary_reduce_kernel(const float *__restrict__ partial, int q_blocks, int blocks, int columns,
                               float *__restrict__ dq_weight, float *__restrict__ dk_weight) {
  __shared__ float sums[32][33];
  heads::await_stream();
  const bool is_key = blockIdx.x & 1;
  const int column0 = blockIdx.x / 2 * 32, column = column0 + threadIdx.x % 32, lane = threadIdx.x / 32;
  const int begin = is_key ? q_blocks : 0, end = is_key ? blocks : q_blocks;
  float total = 0.0f;
  if (column < columns) {
#pragma unroll 4
    for (int row = begin + lane; row < end; row += 32) total += partial[(int64_t)row * columns + column];
  }
  sums[lane][threadIdx.x % 32] = total;
  __syncthreads();
  total = warp_sum(sums[threadIdx.x % 32][lane]);   // warp `lane` now stands for column column0 + lane
  const int result = column0 + lane;
  if (threadIdx.x % 32 == 0 && result < columns) (is_key ? dk_weight : dq_weight)[result] = total;
}

// --------------------------------------------------------------------- host
struct Arguments {
  View3 q, k;
  View1 q_weight, k_weight;
  View2 cosine, sine;
  View1 positions, workspace;
  float epsilon;
  int32_t dtype, interleaved;
};

int check(const char *what, const Arguments &a, const View3 *const *rows, int row_views) {
  if (a.dtype != B200_F32 && a.dtype != B200_F16 && a.dtype != B200_BF16)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", what, a.dtype);
  if (a.interleaved != 0 && a.interleaved != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: interleaved is 0 or 1", what);
  const int size = heads::element_size(a.dtype);
  const int64_t tokens = a.q.d0, columns = a.q.d2;
  for (int i = 0; i < row_views; ++i) {
    const View3 &v = *rows[i];
    if (!heads::sane(v)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
    if (v.d0 != tokens || v.d1 != rows[i % 2]->d1 || v.d2 != columns)
      return fail(B200_ERR_INVALID_ARGUMENT, "%s: the views differ in tokens, heads or columns", what);
  }
  if (columns < 16 || columns > 256 || columns % 16)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: head_dim %lld is not a multiple of 16 in [16, 256]", what, (long long)columns);
  if (tokens >= (int64_t(1) << 31) || a.q.d1 > 65536 || a.k.d1 > 65536)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: 2^31 tokens or more, or more than 65536 heads", what);
  if (a.q_weight.d0 != columns || a.k_weight.d0 != columns)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: a weight does not have head_dim entries", what);
  if (a.cosine.d0 != a.sine.d0 || a.cosine.d1 != a.sine.d1 || a.cosine.d0 < 0 || a.cosine.d1 < 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the cosine and sine tables differ in shape", what);
  if (a.cosine.d1 < 8 || a.cosine.d1 % 8 || 2 * a.cosine.d1 > columns)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: %lld rotated pairs are not a multiple of 8 within head_dim", what, (long long)a.cosine.d1);
  if (a.cosine.d0 >= (int64_t(1) << 31))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the tables have 2^31 rows or more", what);
  if (a.positions.d0 != tokens) return fail(B200_ERR_INVALID_ARGUMENT, "%s: positions does not have one entry a token", what);
  if (!heads::sane(a.positions.d0, a.positions.s0) || !heads::sane(a.cosine.d0, a.cosine.s0) || !heads::sane(a.sine.d0, a.sine.s0))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (!(a.epsilon >= 0.0f) || isinf(a.epsilon)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: epsilon is not a number >= 0", what);
  if (!a.workspace.data || a.workspace.d0 < B200_WORKSPACE_WORDS || a.workspace.s0 != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the workspace needs %d contiguous int32 words", what, B200_WORKSPACE_WORDS);
  for (int i = 0; i < row_views; ++i) {
    const View3 &v = *rows[i];
    if (v.d0 && v.d1 && !v.data) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (v.d0 && v.d1 && !heads::vector_rows(v, size))
      return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                  "%s: rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  }
  if (tokens && (!a.q_weight.data || !a.k_weight.data || !a.positions.data || (a.cosine.d0 && (!a.cosine.data || !a.sine.data))))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (a.q_weight.s0 != 1 || a.k_weight.s0 != 1 || !aligned16(a.q_weight.data) || !aligned16(a.k_weight.data))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: weights need a unit stride and a 16-byte aligned base", what);
  if (!heads::aligned4(a.positions.data) || !heads::aligned4(a.workspace.data))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: positions and workspace are 4-byte aligned", what);
  if (a.cosine.s1 != 1 || a.sine.s1 != 1 || !aligned16(a.cosine.data) || !aligned16(a.sine.data) ||
      (a.cosine.d0 > 1 && (a.cosine.s0 % 4 || a.sine.s0 % 4)))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: tables need a unit inner stride, a 16-byte aligned base and a row pitch of whole 16-byte steps", what);
  return B200_OK;
}

// Whether two views interleave in memory without meeting: rows of one pitch, side by side (slices of one
// fused projection).
bool side_by_side(const View3 &a, const View3 &b, int size) {
  const int64_t gap = ((const char *)b.data - (const char *)a.data) / size;
  if (a.s0 != b.s0 || a.s0 <= 0 || a.s1 <= 0 || b.s1 <= 0) return false;
  if (gap < 0) return side_by_side(b, a, size);
  return gap >= (a.d1 - 1) * a.s1 + a.d2 && gap + (b.d1 - 1) * b.s1 + b.d2 <= a.s0;
}
bool same_view(const View3 &a, const View3 &b) {
  return a.data == b.data && a.d1 == b.d1 && (a.d0 <= 1 || a.s0 == b.s0) && (a.d1 <= 1 || a.s1 == b.s1);
}
bool meet(const View3 &a, const View3 &b, int size) {
  return heads::overlap(heads::span(a, size), heads::span(b, size)) && !side_by_side(a, b, size);
}

// What is written beside rows (the weights' gradients, the scratch and the workspace; `others`), and the outputs' rows against
// what is read beside rows.
int check_beside(const char *what, const Arguments &a, const View3 *const *rows, int count, int size, const heads::Footprint *others,
                 int other_count) {
  using heads::footprint;
  const heads::Footprint read[] = {footprint(a.q_weight, size), footprint(a.k_weight, size), footprint(a.cosine, 4), footprint(a.sine, 4),
                                   footprint(a.positions, 4)};
  const heads::Footprint space = footprint(a.workspace, 4);
  for (int i = 0; i < count; ++i) {
    const heads::Footprint row = footprint(*rows[i], size);
    int status = heads::check_written(what, others, other_count, &row, 1);
    if (status == B200_OK) status = heads::check_written(what, &space, 1, &row, 1);
    if (status == B200_OK && i >= count - 2) status = heads::check_written(what, &row, 1, read, 5);
    if (status != B200_OK) return status;
  }
  const int status = heads::check_written(what, others, other_count, &space, 1);
  return status != B200_OK ? status : heads::check_written(what, others, other_count, read, 5);
}

// Outputs: rows[count - 2] of q and rows[count - 1] of k; before them inputs of q and k in turn.  A row is
// written after it has been read, so an output may BE an input of its own rows, but it meets no other one,
// nor the other output, nor itself.
int check_outputs(const char *what, const View3 *const *rows, int count, int size) {
  const View3 &to_q = *rows[count - 2], &to_k = *rows[count - 1];
  if (!heads::distinct(to_q) || !heads::distinct(to_k)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: an output's elements overlap one another", what);
  if (meet(to_q, to_k, size)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: the outputs overlap", what);
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < count - 2; ++i)
      if (meet(*rows[count - 2 + o], *rows[i], size) && !(i % 2 == o && same_view(*rows[count - 2 + o], *rows[i])))
        return fail(B200_ERR_INVALID_ARGUMENT, "%s: an output overlaps an input that it is not", what);
  return B200_OK;
}

Operand operand(const View3 &x, const View3 *grad, const void *weight, const View3 &out, int rows) {
  Operand o{};
  o.x = x.data;
  o.x_token = x.s0;
  o.x_head = x.s1;
  if (grad) {
    o.grad = grad->data;
    o.grad_token = grad->s0;
    o.grad_head = grad->s1;
  }
  o.weight = weight;
  o.out = const_cast<void *>(out.data);
  o.out_token = out.s0;
  o.out_head = out.s1;
  o.heads = (int)x.d1;
  o.slices = (uint32_t)((x.d1 + rows - 1) / rows);
  return o;
}

Rotation rotation(const Arguments &a) {
  Rotation r{};
  r.cosine = static_cast<const float *>(a.cosine.data);
  r.sine = static_cast<const float *>(a.sine.data);
  r.cosine_row = a.cosine.s0;
  r.sine_row = a.sine.s0;
  r.table_rows = (int)a.cosine.d0;
  r.half = (int)a.cosine.d1;
  r.columns = (int)a.q.d2;
  r.interleaved = a.interleaved;
  r.positions = static_cast<const int *>(a.positions.data);
  r.positions_step = a.positions.s0;
  r.tokens = (int)a.q.d0;
  r.inverse_columns = 1.0f / (float)a.q.d2;
  r.epsilon = a.epsilon;
  r.status = static_cast<int *>(const_cast<void *>(a.workspace.data));
  return r;
}

// Heads of a token that a unit takes: as many as leave every resident group of lanes some work, at most
// 8 (one load of the angles is then a tenth of what the rows move), and so that no more than a seventh of
// the rounds fall on rows that are not there.
int rows_of_unit(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t columns) {
  const int64_t groups = (int64_t)kBlocksPerSm * sm_count() * kThreads / heads::row_lanes(columns), all = q_heads + k_heads;
  for (int64_t rows = 8; rows > 1; --rows) {
    const int64_t units = (q_heads + rows - 1) / rows + (k_heads + rows - 1) / rows;
    if (tokens * units >= groups && units * rows * 7 <= all * 8) return (int)rows;
  }
  return 1;
}

template <typename T, int LANES>
int launch_forward(const Operand &q, const Operand &k, const Rotation &r, int unit_rows, cudaStream_t stream) {
  constexpr int kBytes = Ring<2 * Eight<T>::kVectors, kForwardStages<T>>::kBytes, kGroups = kThreads / LANES;
  const auto kernel = head_norm_rotary_kernel<T, LANES>;
  B200_CUDA_TRY(opt_in_dynamic_smem(kernel, kBytes));
  const int64_t units = (int64_t)r.tokens * (q.slices + k.slices), need = (units + kGroups - 1) / kGroups;
  const int64_t resident = (int64_t)kBlocksPerSm * sm_count();
  B200_CUDA_TRY(heads::launch_early(kernel, (unsigned)(need < resident ? need : resident), kThreads, kBytes, stream, q, k, r, unit_rows,
                                    (uint32_t)units));
  return B200_OK;
}

template <typename T> int forward(const Arguments &a, const View3 &q_out, const View3 &k_out, cudaStream_t stream) {
  const int unit_rows = rows_of_unit(a.q.d0, a.q.d1, a.k.d1, a.q.d2);
  const Operand q = operand(a.q, nullptr, a.q_weight.data, q_out, unit_rows), k = operand(a.k, nullptr, a.k_weight.data, k_out, unit_rows);
  const int status = heads::check_units("head_norm_rotary", a.q.d0, (int64_t)q.slices + k.slices);
  if (status != B200_OK) return status;
  const Rotation r = rotation(a);
  switch (heads::row_lanes(r.columns)) {
  case 1: return launch_forward<T, 1>(q, k, r, unit_rows, stream);
  case 2: return launch_forward<T, 2>(q, k, r, unit_rows, stream);
  case 4: return launch_forward<T, 4>(q, k, r, unit_rows, stream);
  case 8: return launch_forward<T, 8>(q, k, r, unit_rows, stream);
  default: return launch_forward<T, 16>(q, k, r, unit_rows, stream);
  }
}

// Blocks of the backward pass: as many as are resident at once, q's and k's in proportion to their rows.
struct BackwardShape {
  int unit_rows, q_blocks, blocks;
};
BackwardShape backward_shape(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t columns) {
  const int unit_rows = rows_of_unit(tokens, q_heads, k_heads, columns);
  const int64_t groups = kThreads / heads::row_lanes(columns);
  const auto need = [&](int64_t heads) { return (tokens * ((heads + unit_rows - 1) / unit_rows) + groups - 1) / groups; };
  const int64_t most = (int64_t)kBlocksPerSm * sm_count(), q_need = need(q_heads), k_need = need(k_heads);
  int64_t q_blocks = q_need, k_blocks = k_need;
  if (q_need + k_need > most) {
    q_blocks = most * q_need / (q_need + k_need);
    if (q_blocks < 1 && q_need) q_blocks = 1;
    k_blocks = most - q_blocks;
    if (k_blocks < 1 && k_need) { k_blocks = 1; q_blocks = most - 1; }
  }
  return {unit_rows, (int)q_blocks, (int)(q_blocks + k_blocks)};
}

template <typename T, int LANES>
cudaError_t launch_backward(const Operand &q, const Operand &k, const Rotation &r, const BackwardShape &shape, float *partial,
                            cudaStream_t stream) {
  if (!shape.blocks) return cudaSuccess;
  constexpr int kBytes = Ring<4 * Eight<T>::kVectors, kBackwardStages<T>>::kBytes;
  const auto kernel = head_norm_rotary_backward_kernel<T, LANES>;
  const cudaError_t error = opt_in_dynamic_smem(kernel, kBytes);
  if (error != cudaSuccess) return error;
  return heads::launch_early(kernel, shape.blocks, kThreads, kBytes, stream, q, k, r, shape.unit_rows, shape.q_blocks, partial);
}

template <typename T>
int backward(const Arguments &a, const View3 &grad_q, const View3 &grad_k, const View3 &dq, const View3 &dk, float *partial,
             float *dq_weight, float *dk_weight, cudaStream_t stream) {
  const BackwardShape shape = backward_shape(a.q.d0, a.q.d1, a.k.d1, a.q.d2);
  const Operand q = operand(a.q, &grad_q, a.q_weight.data, dq, shape.unit_rows);
  const Operand k = operand(a.k, &grad_k, a.k_weight.data, dk, shape.unit_rows);
  const int status = heads::check_units("head_norm_rotary_backward", a.q.d0, (int64_t)q.slices + k.slices);
  if (status != B200_OK) return status;
  const Rotation r = rotation(a);
  cudaError_t error;
  switch (heads::row_lanes(r.columns)) {
  case 1: error = launch_backward<T, 1>(q, k, r, shape, partial, stream); break;
  case 2: error = launch_backward<T, 2>(q, k, r, shape, partial, stream); break;
  case 4: error = launch_backward<T, 4>(q, k, r, shape, partial, stream); break;
  case 8: error = launch_backward<T, 8>(q, k, r, shape, partial, stream); break;
  default: error = launch_backward<T, 16>(q, k, r, shape, partial, stream); break;
  }
  if (error != cudaSuccess) return cuda_fail(error, "head_norm_rotary_backward");
  B200_CUDA_TRY(heads::launch_early(head_norm_rotary_reduce_kernel, 2 * ((r.columns + 31) / 32), 1024, 0, stream, partial,
                                    shape.q_blocks, shape.blocks, r.columns, dq_weight, dk_weight));
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_head_norm_rotary(const int64_t *slots, int64_t count, float epsilon, int32_t dtype, int32_t interleaved,
                                     void *stream) {
  const char *what = "head_norm_rotary";
  heads::Slots from(slots, count);
  Arguments a{};
  a.q = from.view3();
  a.k = from.view3();
  a.q_weight = from.view1();
  a.k_weight = from.view1();
  a.cosine = from.view2();
  a.sine = from.view2();
  a.positions = from.view1();
  const View3 to_q = from.view3(), to_k = from.view3();
  a.workspace = from.view1();
  if (!from.exact()) return fail(B200_ERR_INVALID_ARGUMENT, "%s: %lld slots do not describe its views", what, (long long)count);
  a.epsilon = epsilon;
  a.dtype = dtype;
  a.interleaved = interleaved;
  const View3 *const rows[] = {&a.q, &a.k, &to_q, &to_k};
  int status = check(what, a, rows, 4);
  if (status != B200_OK) return status;
  if (a.q.d0 == 0 || a.q.d1 + a.k.d1 == 0) return B200_OK;
  const int size = heads::element_size(dtype);
  status = check_outputs(what, rows, 4, size);
  if (status == B200_OK) status = check_beside(what, a, rows, 4, size, nullptr, 0);
  if (status != B200_OK) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
  case B200_F32: return forward<float>(a, to_q, to_k, s);
  case B200_F16: return forward<__half>(a, to_q, to_k, s);
  default: return forward<__nv_bfloat16>(a, to_q, to_k, s);
  }
}

extern "C" int b200_head_norm_rotary_scratch(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t head_dim, int64_t *rows) {
  if (!rows || tokens < 0 || q_heads < 0 || k_heads < 0 || tokens >= (int64_t(1) << 31) || q_heads > 65536 || k_heads > 65536 ||
      head_dim < 1 || head_dim > 256)
    return fail(B200_ERR_INVALID_ARGUMENT, "head_norm_rotary_scratch: an extent is out of range");
  *rows = backward_shape(tokens, q_heads, k_heads, head_dim).blocks;
  return B200_OK;
}

extern "C" int b200_head_norm_rotary_backward(const int64_t *slots, int64_t count, float epsilon, int32_t dtype,
                                              int32_t interleaved, void *stream) {
  const char *what = "head_norm_rotary_backward";
  heads::Slots from(slots, count);
  Arguments a{};
  const View3 from_q = from.view3(), from_k = from.view3();
  a.q = from.view3();
  a.k = from.view3();
  a.q_weight = from.view1();
  a.k_weight = from.view1();
  a.cosine = from.view2();
  a.sine = from.view2();
  a.positions = from.view1();
  const View3 to_q = from.view3(), to_k = from.view3();
  const View1 to_q_weight = from.view1(), to_k_weight = from.view1();
  const View2 partial = from.view2();
  a.workspace = from.view1();
  if (!from.exact()) return fail(B200_ERR_INVALID_ARGUMENT, "%s: %lld slots do not describe its views", what, (long long)count);
  a.epsilon = epsilon;
  a.dtype = dtype;
  a.interleaved = interleaved;
  const View3 *const rows[] = {&a.q, &a.k, &from_q, &from_k, &to_q, &to_k};
  int status = check(what, a, rows, 6);
  if (status != B200_OK) return status;
  if (!to_q_weight.data || !to_k_weight.data || to_q_weight.d0 != a.q.d2 || to_k_weight.d0 != a.q.d2)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: a weight's gradient does not have head_dim entries", what);
  if (to_q_weight.s0 != 1 || to_k_weight.s0 != 1 || !heads::aligned4(to_q_weight.data) || !heads::aligned4(to_k_weight.data))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the weights' gradients need a unit stride and 4-byte alignment", what);
  const BackwardShape shape = backward_shape(a.q.d0, a.q.d1, a.k.d1, a.q.d2);
  if (partial.d0 < shape.blocks || partial.d1 != a.q.d2 || (shape.blocks && !partial.data))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the scratch needs (%d, head_dim) f32", what, shape.blocks);
  if (!heads::aligned4(partial.data) || partial.s1 != 1 || (shape.blocks > 1 && partial.s0 != partial.d1))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the scratch is contiguous and 4-byte aligned", what);
  const int size = heads::element_size(dtype);
  status = check_outputs(what, rows, 6, size);
  const heads::Footprint others[] = {heads::footprint(to_q_weight, 4), heads::footprint(to_k_weight, 4), heads::footprint(partial, 4)};
  if (status == B200_OK) status = check_beside(what, a, rows, 6, size, others, 3);
  if (status != B200_OK) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float *scratch = static_cast<float *>(const_cast<void *>(partial.data));
  float *dqw = static_cast<float *>(const_cast<void *>(to_q_weight.data)), *dkw = static_cast<float *>(const_cast<void *>(to_k_weight.data));
  switch (dtype) {
  case B200_F32: return backward<float>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  case B200_F16: return backward<__half>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  default: return backward<__nv_bfloat16>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  }
}
