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
#include "heads.cuh"

namespace b200 {
namespace {

using heads::Eight;
using heads::View3;

constexpr int kThreads = 256;

struct Operand {        // one of q, k (and, for the backward pass, its gradients)
  const void *x;
  const void *grad;     // backward only
  const void *weight;
  void *out;
  int64_t x_token, x_head, grad_token, grad_head, out_token, out_head;
  int heads;
  int slices;           // units per token: ceil(heads / rows of a unit)
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

// x[0..8) and x[8..16) are the pieces; BACK turns by the opposite angle.
template <bool BACK>
__device__ __forceinline__ void turn(float (&x)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1], t = BACK ? -s[i] : s[i];
      x[2 * i] = a * c[i] - b * t;
      x[2 * i + 1] = b * c[i] + a * t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i], b = x[i + 8], t = BACK ? -s[i] : s[i];
      x[i] = a * c[i] - b * t;
      x[i + 8] = b * c[i] + a * t;
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

// ------------------------------------------------------------------ forward
// A unit is ROWS heads of one token, all of q or all of k: ROWS x 2 vectors in flight in a lane.
template <typename T, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads)
head_norm_rotary_kernel(Operand q, Operand k, Rotation r) {
  const int e = threadIdx.x % LANES;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int slices = q.slices + k.slices;
  const int token = (int)(unit / slices);
  const bool unit_live = token < r.tokens;
  int slice = (int)(unit - (int64_t)token * slices);
  const bool is_key = slice >= q.slices;
  if (is_key) slice -= q.slices;
  const int head_count = is_key ? k.heads : q.heads;
  const int head0 = slice * ROWS;
  const bool lane_live = unit_live && e * 16 < r.columns;
  int first, second;
  pieces(r, e, first, second);

  Eight<T> a[ROWS], b[ROWS];
  const T *source = static_cast<const T *>(is_key ? k.x : q.x) +
                    (unit_live ? token * (is_key ? k.x_token : q.x_token) : 0);
  const int64_t source_head = is_key ? k.x_head : q.x_head;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    a[i].clear();
    b[i].clear();
    if (lane_live && head0 + i < head_count) {
      a[i].load(source + (head0 + i) * source_head + first);
      b[i].load(source + (head0 + i) * source_head + second);
    }
  }
  const int position = unit_live ? place(r, token, e == 0) : -1;
  const bool turned = lane_live && e * 8 < r.half && position >= 0;
  float cosine[8], sine[8];
  if (turned) {
    const float4 *c4 = reinterpret_cast<const float4 *>(r.cosine + position * r.cosine_row + 8 * e);
    const float4 *s4 = reinterpret_cast<const float4 *>(r.sine + position * r.sine_row + 8 * e);
    const float4 c0 = __ldg(c4), c1 = __ldg(c4 + 1), s0 = __ldg(s4), s1 = __ldg(s4 + 1);
    cosine[0] = c0.x; cosine[1] = c0.y; cosine[2] = c0.z; cosine[3] = c0.w;
    cosine[4] = c1.x; cosine[5] = c1.y; cosine[6] = c1.z; cosine[7] = c1.w;
    sine[0] = s0.x; sine[1] = s0.y; sine[2] = s0.z; sine[3] = s0.w;
    sine[4] = s1.x; sine[5] = s1.y; sine[6] = s1.z; sine[7] = s1.w;
  }
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = 0.0f;
  if (lane_live) {
    const T *weight = static_cast<const T *>(is_key ? k.weight : q.weight);
    Eight<T> w0, w1;
    w0.load(weight + first);
    w1.load(weight + second);
    w0.widen(w);
    w1.widen(w + 8);
  }
  T *target = static_cast<T *>(is_key ? k.out : q.out) + (unit_live ? token * (is_key ? k.out_token : q.out_token) : 0);
  const int64_t target_head = is_key ? k.out_head : q.out_head;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float x[16];
    a[i].widen(x);
    b[i].widen(x + 8);
    float squares = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) squares += x[j] * x[j];
    squares = heads::row_sum<LANES>(squares);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(squares * r.inverse_columns + r.epsilon));
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = position < 0 ? 0.0f : x[j] * rstd * w[j];
    if (turned) turn<false>(x, cosine, sine, r.interleaved);   // other columns pass as they are, infinities too
    if (lane_live && head0 + i < head_count) {
      a[i].narrow(x);
      b[i].narrow(x + 8);
      a[i].store(target + (head0 + i) * target_head + first);
      b[i].store(target + (head0 + i) * target_head + second);
    }
  }
}

// ----------------------------------------------------------------- backward
// The blocks of [0, q_blocks) take q's units, the others k's, so that a lane keeps the sums of one
// weight only: 16 columns in f32, over all the rows it meets.  A block adds its lanes' sums in a
// fixed order and writes one row of `partial`; the second kernel adds those rows, again in a fixed
// order, so that dw does not vary from run to run.
constexpr int kUnitRows = 8;   // heads of a token that share one load of its cosines and sines

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads)
head_norm_rotary_backward_kernel(Operand q, Operand k, Rotation r, int q_blocks, float *__restrict__ partial) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float sums[kGroups][LANES * 16 + 1];
  const int e = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool is_key = (int)blockIdx.x >= q_blocks;
  const Operand &o = is_key ? k : q;
  const int block = is_key ? blockIdx.x - q_blocks : blockIdx.x;
  const int blocks = is_key ? gridDim.x - q_blocks : q_blocks;
  const bool lane_live = e * 16 < r.columns;
  int first, second;
  pieces(r, e, first, second);
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = dw[i] = 0.0f;
  if (lane_live) {
    const T *weight = static_cast<const T *>(o.weight);
    Eight<T> w0, w1;
    w0.load(weight + first);
    w1.load(weight + second);
    w0.widen(w);
    w1.widen(w + 8);
  }
  const int64_t units = (int64_t)r.tokens * o.slices;
  // every group of the block runs the same number of rounds: the shuffles below are whole-warp
  for (int64_t base = (int64_t)block * kGroups; base < units; base += (int64_t)blocks * kGroups) {
    const int64_t unit = base + group;
    const bool unit_live = unit < units;
    const int token = unit_live ? (int)(unit / o.slices) : 0;
    const int head0 = unit_live ? (int)(unit - (int64_t)token * o.slices) * kUnitRows : 0;
    const int rows = unit_live ? min(kUnitRows, o.heads - head0) : 0;
    const int position = unit_live ? place(r, token, e == 0) : -1;
    const bool turned = lane_live && e * 8 < r.half && position >= 0;
    float cosine[8], sine[8];
    if (turned) {
      const float *c = r.cosine + position * r.cosine_row + 8 * e, *s = r.sine + position * r.sine_row + 8 * e;
#pragma unroll
      for (int i = 0; i < 8; ++i) { cosine[i] = __ldg(c + i); sine[i] = __ldg(s + i); }
    }
    const T *x_row = static_cast<const T *>(o.x) + token * o.x_token + head0 * o.x_head;
    const T *grad_row = static_cast<const T *>(o.grad) + token * o.grad_token + head0 * o.grad_head;
    T *out_row = static_cast<T *>(o.out) + token * o.out_token + head0 * o.out_head;
#pragma unroll 2
    for (int row = 0; row < kUnitRows; ++row) {
      const bool live = lane_live && row < rows;
      Eight<T> xa, xb, ga, gb;
      xa.clear(); xb.clear(); ga.clear(); gb.clear();
      if (live && position >= 0) {
        xa.load(x_row + row * o.x_head + first);
        xb.load(x_row + row * o.x_head + second);
        ga.load(grad_row + row * o.grad_head + first);
        gb.load(grad_row + row * o.grad_head + second);
      }
      float x[16], g[16];
      xa.widen(x); xb.widen(x + 8);
      ga.widen(g); gb.widen(g + 8);
      float squares = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) squares += x[j] * x[j];
      squares = heads::row_sum<LANES>(squares);
      const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(squares * r.inverse_columns + r.epsilon));
      if (turned) turn<true>(g, cosine, sine, r.interleaved);
      float projection = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] *= rstd;
        dw[j] += g[j] * x[j];
        g[j] *= w[j];
        projection += g[j] * x[j];
      }
      projection = heads::row_sum<LANES>(projection) * r.inverse_columns;
      if (live) {
#pragma unroll
        for (int j = 0; j < 16; ++j) g[j] = position < 0 ? 0.0f : rstd * (g[j] - x[j] * projection);
        xa.narrow(g);
        xb.narrow(g + 8);
        xa.store(out_row + row * o.out_head + first);
        xb.store(out_row + row * o.out_head + second);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) sums[group][i * LANES + e] = dw[i];
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

// 32 columns x 32 lanes of rows: blockIdx.y 0 adds q's rows of `partial`, 1 adds k's.
__global__ void __launch_bounds__(1024)
head_norm_rotary_reduce_kernel(const float *__restrict__ partial, int q_blocks, int blocks, int columns,
                               float *__restrict__ dq_weight, float *__restrict__ dk_weight) {
  __shared__ float sums[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int column = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  const int begin = blockIdx.y ? q_blocks : 0, end = blockIdx.y ? blocks : q_blocks;
  float total = 0.0f;
  if (column < columns) {
#pragma unroll 4
    for (int row = begin + lane; row < end; row += 32) total += partial[(int64_t)row * columns + column];
  }
  sums[lane][threadIdx.x % 32] = total;
  __syncthreads();
  total = warp_sum(sums[threadIdx.x % 32][lane]);   // lane `lane` of the block now stands for column blockIdx.x * 32 + lane
  const int result = blockIdx.x * 32 + lane;
  if (threadIdx.x % 32 == 0 && result < columns) (blockIdx.y ? dk_weight : dq_weight)[result] = total;
}

// --------------------------------------------------------------------- host
struct Arguments {
  View3 q, k;
  const void *q_weight, *k_weight;
  int64_t q_weight_d0, q_weight_s0, k_weight_d0, k_weight_s0;
  const void *cosine, *sine;
  int64_t cos_d0, cos_d1, cos_s0, cos_s1, sin_d0, sin_d1, sin_s0, sin_s1;
  const void *positions;
  int64_t positions_d0, positions_s0;
  float epsilon;
  void *workspace;
  int64_t ws_d0, ws_s0;
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
  if (a.q_weight_d0 != columns || a.k_weight_d0 != columns)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: a weight does not have head_dim entries", what);
  if (a.cos_d0 != a.sin_d0 || a.cos_d1 != a.sin_d1 || a.cos_d0 < 0 || a.cos_d1 < 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the cosine and sine tables differ in shape", what);
  if (a.cos_d1 < 8 || a.cos_d1 % 8 || 2 * a.cos_d1 > columns)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: %lld rotated pairs are not a multiple of 8 within head_dim", what, (long long)a.cos_d1);
  if (a.cos_d0 >= (int64_t(1) << 31))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the tables have 2^31 rows or more", what);
  if (a.positions_d0 != tokens) return fail(B200_ERR_INVALID_ARGUMENT, "%s: positions does not have one entry a token", what);
  if (!heads::sane(a.positions_d0, a.positions_s0) || !heads::sane(a.cos_d0, a.cos_s0) || !heads::sane(a.sin_d0, a.sin_s0))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (!(a.epsilon >= 0.0f) || isinf(a.epsilon)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: epsilon is not a number >= 0", what);
  if (!a.workspace || a.ws_d0 < B200_WORKSPACE_WORDS || a.ws_s0 != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the workspace needs %d contiguous int32 words", what, B200_WORKSPACE_WORDS);
  for (int i = 0; i < row_views; ++i) {
    const View3 &v = *rows[i];
    if (v.d0 && v.d1 && !v.data) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (v.d0 && v.d1 && !heads::vector_rows(v, size))
      return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                  "%s: rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  }
  if (tokens && (!a.q_weight || !a.k_weight || !a.positions || (a.cos_d0 && (!a.cosine || !a.sine))))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (a.q_weight_s0 != 1 || a.k_weight_s0 != 1 || !aligned16(a.q_weight) || !aligned16(a.k_weight))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: weights need a unit stride and a 16-byte aligned base", what);
  if (a.cos_s1 != 1 || a.sin_s1 != 1 || !aligned16(a.cosine) || !aligned16(a.sine) ||
      (a.cos_d0 > 1 && (a.cos_s0 % 4 || a.sin_s0 % 4)))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: tables need a unit inner stride, a 16-byte aligned base and a row pitch of whole 16-byte steps", what);
  return B200_OK;
}

// An output is written row by row after the row has been read: it may BE an input view (same base
// and strides), but may not overlap one in any other way, nor another output.
int check_output(const char *what, const View3 &out, int size, const View3 *const *inputs, int count, const View3 *other) {
  if (!heads::distinct(out)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: an output's elements overlap one another", what);
  const heads::Span span = heads::span(out, size);
  for (int i = 0; i < count; ++i) {
    const View3 &in = *inputs[i];
    const bool same = in.data == out.data && in.d1 == out.d1 && (in.d0 <= 1 || in.s0 == out.s0) && (in.d1 <= 1 || in.s1 == out.s1);
    // two views of one fused projection interleave in memory: rows of the same pitch that never meet
    const int64_t gap = ((const char *)in.data - (const char *)out.data) / size;
    const int64_t pitch = out.s0;
    const bool aside = !same && in.s0 == pitch && pitch > 0 && in.s1 > 0 && out.s1 > 0 &&
                       ((gap > 0 && gap >= (out.d1 - 1) * out.s1 + out.d2 && gap + (in.d1 - 1) * in.s1 + in.d2 <= pitch) ||
                        (gap < 0 && -gap >= (in.d1 - 1) * in.s1 + in.d2 && -gap + (out.d1 - 1) * out.s1 + out.d2 <= pitch));
    if (!same && !aside && heads::overlap(span, heads::span(in, size)))
      return fail(B200_ERR_INVALID_ARGUMENT, "%s: an output overlaps an input that it is not", what);
  }
  if (other) {
    const View3 *const one[] = {other};
    const bool same = other->data == out.data && out.d0 && out.d1 && other->d1;
    if (same) return fail(B200_ERR_INVALID_ARGUMENT, "%s: the outputs overlap", what);
    return check_output(what, out, size, one, 1, nullptr);
  }
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
  o.slices = (int)((x.d1 + rows - 1) / rows);
  return o;
}

Rotation rotation(const Arguments &a) {
  Rotation r{};
  r.cosine = static_cast<const float *>(a.cosine);
  r.sine = static_cast<const float *>(a.sine);
  r.cosine_row = a.cos_s0;
  r.sine_row = a.sin_s0;
  r.table_rows = (int)a.cos_d0;
  r.half = (int)a.cos_d1;
  r.columns = (int)a.q.d2;
  r.interleaved = a.interleaved;
  r.positions = static_cast<const int *>(a.positions);
  r.positions_step = a.positions_s0;
  r.tokens = (int)a.q.d0;
  r.inverse_columns = 1.0f / (float)a.q.d2;
  r.epsilon = a.epsilon;
  r.status = static_cast<int *>(a.workspace);
  return r;
}

template <typename T, int ROWS> int launch_forward(const Arguments &a, const View3 &q_out, const View3 &k_out, cudaStream_t stream) {
  const Operand q = operand(a.q, nullptr, a.q_weight, q_out, ROWS), k = operand(a.k, nullptr, a.k_weight, k_out, ROWS);
  const Rotation r = rotation(a);
  const int lanes = heads::row_lanes(r.columns);
  const int64_t units = (int64_t)r.tokens * (q.slices + k.slices), per_block = kThreads / lanes;
  const int64_t blocks = (units + per_block - 1) / per_block;
  if (blocks >= (int64_t(1) << 31)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "head_norm_rotary: too many rows for one launch");
  switch (lanes) {
  case 1: head_norm_rotary_kernel<T, 1, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(q, k, r); break;
  case 2: head_norm_rotary_kernel<T, 2, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(q, k, r); break;
  case 4: head_norm_rotary_kernel<T, 4, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(q, k, r); break;
  case 8: head_norm_rotary_kernel<T, 8, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(q, k, r); break;
  default: head_norm_rotary_kernel<T, 16, ROWS><<<(unsigned)blocks, kThreads, 0, stream>>>(q, k, r); break;
  }
  B200_CUDA_TRY(cudaGetLastError());
  return B200_OK;
}

template <typename T> int forward(const Arguments &a, const View3 &q_out, const View3 &k_out, cudaStream_t stream) {
  return launch_forward<T, 1>(a, q_out, k_out, stream);
}

// Blocks of the backward pass: as many as are resident at once, q's and k's in proportion to their rows.
struct BackwardShape {
  int q_blocks, blocks;
};
BackwardShape backward_shape(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t columns) {
  const int64_t groups = kThreads / heads::row_lanes(columns);
  const auto need = [&](int64_t heads) {
    return (tokens * ((heads + kUnitRows - 1) / kUnitRows) + groups - 1) / groups;
  };
  const int64_t most = 3 * (int64_t)sm_count(), q_need = need(q_heads), k_need = need(k_heads);
  int64_t q_blocks = q_need, k_blocks = k_need;
  if (q_need + k_need > most) {
    q_blocks = most * q_need / (q_need + k_need);
    if (q_blocks < 1 && q_need) q_blocks = 1;
    k_blocks = most - q_blocks;
    if (k_blocks < 1 && k_need) { k_blocks = 1; q_blocks = most - 1; }
  }
  return {(int)q_blocks, (int)(q_blocks + k_blocks)};
}

template <typename T, int LANES>
cudaError_t launch_backward(const Operand &q, const Operand &k, const Rotation &r, const BackwardShape &shape, float *partial,
                            cudaStream_t stream) {
  if (shape.blocks)
    head_norm_rotary_backward_kernel<T, LANES><<<shape.blocks, kThreads, 0, stream>>>(q, k, r, shape.q_blocks, partial);
  return cudaGetLastError();
}

template <typename T>
int backward(const Arguments &a, const View3 &grad_q, const View3 &grad_k, const View3 &dq, const View3 &dk, float *partial,
             float *dq_weight, float *dk_weight, cudaStream_t stream) {
  const Operand q = operand(a.q, &grad_q, a.q_weight, dq, kUnitRows), k = operand(a.k, &grad_k, a.k_weight, dk, kUnitRows);
  const Rotation r = rotation(a);
  const BackwardShape shape = backward_shape(a.q.d0, a.q.d1, a.k.d1, a.q.d2);
  cudaError_t error;
  switch (heads::row_lanes(r.columns)) {
  case 1: error = launch_backward<T, 1>(q, k, r, shape, partial, stream); break;
  case 2: error = launch_backward<T, 2>(q, k, r, shape, partial, stream); break;
  case 4: error = launch_backward<T, 4>(q, k, r, shape, partial, stream); break;
  case 8: error = launch_backward<T, 8>(q, k, r, shape, partial, stream); break;
  default: error = launch_backward<T, 16>(q, k, r, shape, partial, stream); break;
  }
  if (error != cudaSuccess) return cuda_fail(error, "head_norm_rotary_backward");
  // the reduction is placed while the first kernel still runs and waits for its end on the device
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((r.columns + 31) / 32, 2);
  config.blockDim = dim3(1024);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = shape.blocks ? 1 : 0;
  B200_CUDA_TRY(cudaLaunchKernelEx(&config, head_norm_rotary_reduce_kernel, (const float *)partial, shape.q_blocks, shape.blocks,
                                   r.columns, dq_weight, dk_weight));
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

#define VIEW3(name) \
  View3 { name, name##_d0, name##_d1, name##_d2, name##_s0, name##_s1, name##_s2 }
#define ARGUMENTS                                                                                                        \
  Arguments {                                                                                                            \
    VIEW3(q), VIEW3(k), q_weight, k_weight, q_weight_d0, q_weight_s0, k_weight_d0, k_weight_s0, cosine, sine, cosine_d0, \
        cosine_d1, cosine_s0, cosine_s1, sine_d0, sine_d1, sine_s0, sine_s1, positions, positions_d0, positions_s0,      \
        epsilon, workspace, ws_d0, ws_s0, dtype, interleaved                                                             \
  }

extern "C" int b200_head_norm_rotary(
    const void *q, int64_t q_d0, int64_t q_d1, int64_t q_d2, int64_t q_s0, int64_t q_s1, int64_t q_s2,
    const void *k, int64_t k_d0, int64_t k_d1, int64_t k_d2, int64_t k_s0, int64_t k_s1, int64_t k_s2,
    const void *q_weight, int64_t q_weight_d0, int64_t q_weight_s0,
    const void *k_weight, int64_t k_weight_d0, int64_t k_weight_s0,
    const void *cosine, int64_t cosine_d0, int64_t cosine_d1, int64_t cosine_s0, int64_t cosine_s1,
    const void *sine, int64_t sine_d0, int64_t sine_d1, int64_t sine_s0, int64_t sine_s1,
    const void *positions, int64_t positions_d0, int64_t positions_s0,
    void *q_out, int64_t q_out_d0, int64_t q_out_d1, int64_t q_out_d2, int64_t q_out_s0, int64_t q_out_s1, int64_t q_out_s2,
    void *k_out, int64_t k_out_d0, int64_t k_out_d1, int64_t k_out_d2, int64_t k_out_s0, int64_t k_out_s1, int64_t k_out_s2,
    float epsilon, void *workspace, int64_t ws_d0, int64_t ws_s0, int32_t dtype, int32_t interleaved, void *stream) {
  const char *what = "head_norm_rotary";
  const Arguments a = ARGUMENTS;
  const View3 to_q = VIEW3(q_out), to_k = VIEW3(k_out);
  const View3 *const rows[] = {&a.q, &a.k, &to_q, &to_k};
  int status = check(what, a, rows, 4);
  if (status != B200_OK) return status;
  if (a.q.d0 == 0 || a.q.d1 + a.k.d1 == 0) return B200_OK;
  const int size = heads::element_size(dtype);
  status = check_output(what, to_q, size, rows, 2, &to_k);
  if (status == B200_OK) status = check_output(what, to_k, size, rows, 2, nullptr);
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

extern "C" int b200_head_norm_rotary_backward(
    const void *grad_q, int64_t grad_q_d0, int64_t grad_q_d1, int64_t grad_q_d2, int64_t grad_q_s0, int64_t grad_q_s1, int64_t grad_q_s2,
    const void *grad_k, int64_t grad_k_d0, int64_t grad_k_d1, int64_t grad_k_d2, int64_t grad_k_s0, int64_t grad_k_s1, int64_t grad_k_s2,
    const void *q, int64_t q_d0, int64_t q_d1, int64_t q_d2, int64_t q_s0, int64_t q_s1, int64_t q_s2,
    const void *k, int64_t k_d0, int64_t k_d1, int64_t k_d2, int64_t k_s0, int64_t k_s1, int64_t k_s2,
    const void *q_weight, int64_t q_weight_d0, int64_t q_weight_s0,
    const void *k_weight, int64_t k_weight_d0, int64_t k_weight_s0,
    const void *cosine, int64_t cosine_d0, int64_t cosine_d1, int64_t cosine_s0, int64_t cosine_s1,
    const void *sine, int64_t sine_d0, int64_t sine_d1, int64_t sine_s0, int64_t sine_s1,
    const void *positions, int64_t positions_d0, int64_t positions_s0,
    void *dq, int64_t dq_d0, int64_t dq_d1, int64_t dq_d2, int64_t dq_s0, int64_t dq_s1, int64_t dq_s2,
    void *dk, int64_t dk_d0, int64_t dk_d1, int64_t dk_d2, int64_t dk_s0, int64_t dk_s1, int64_t dk_s2,
    void *dq_weight, int64_t dq_weight_d0, int64_t dq_weight_s0, void *dk_weight, int64_t dk_weight_d0, int64_t dk_weight_s0,
    void *partial, int64_t partial_d0, int64_t partial_d1, int64_t partial_s0, int64_t partial_s1,
    float epsilon, void *workspace, int64_t ws_d0, int64_t ws_s0, int32_t dtype, int32_t interleaved, void *stream) {
  const char *what = "head_norm_rotary_backward";
  const Arguments a = ARGUMENTS;
  const View3 from_q = VIEW3(grad_q), from_k = VIEW3(grad_k), to_q = VIEW3(dq), to_k = VIEW3(dk);
  const View3 *const rows[] = {&a.q, &a.k, &from_q, &from_k, &to_q, &to_k};
  int status = check(what, a, rows, 6);
  if (status != B200_OK) return status;
  if (!dq_weight || !dk_weight || dq_weight_d0 != a.q.d2 || dk_weight_d0 != a.q.d2)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: a weight's gradient does not have head_dim entries", what);
  if (dq_weight_s0 != 1 || dk_weight_s0 != 1)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the weights' gradients need a unit stride", what);
  const BackwardShape shape = backward_shape(a.q.d0, a.q.d1, a.k.d1, a.q.d2);
  if (partial_d0 < shape.blocks || partial_d1 != a.q.d2 || (shape.blocks && !partial))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the scratch needs (%d, head_dim) f32", what, shape.blocks);
  if (partial_s1 != 1 || (shape.blocks > 1 && partial_s0 != partial_d1))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: the scratch is contiguous", what);
  const int size = heads::element_size(dtype);
  status = check_output(what, to_q, size, rows, 4, &to_k);
  if (status == B200_OK) status = check_output(what, to_k, size, rows, 4, nullptr);
  if (status != B200_OK) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float *scratch = static_cast<float *>(partial), *dqw = static_cast<float *>(dq_weight), *dkw = static_cast<float *>(dk_weight);
  switch (dtype) {
  case B200_F32: return backward<float>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  case B200_F16: return backward<__half>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  default: return backward<__nv_bfloat16>(a, from_q, from_k, to_q, to_k, scratch, dqw, dkw, s);
  }
}
