// Attention of one new token a sequence over a paged key-value cache in 16 or 8 bits.
//
//     s_j = scale (q . k_j)      out = sum_j e^(s_j) v_j / sum_j e^(s_j)      lse = log sum_j e^(s_j)
//
// The cache is read once and is nearly all that is read, so HBM bounds it: 4 D bytes (16 bits) or
// 2 D + 8 (8 bits) for a key position of a head, against 4 D operations for each of the `group` query
// heads that share it.  What the kernel has to do is keep copies in flight on every SM, whatever
// the lengths are.
//
// Work.  The unit is a step: WARPS * KEYS key positions of one (sequence, key head, row tile).  All
// steps of the call, sequence after sequence, are cut into as many equal runs as there are resident
// blocks; a block finds its run by a scan of the lengths and crosses from one sequence to the next
// without draining its copies.  A ragged batch therefore loads all SMs alike, a single long
// sequence is spread over all of them, and a short one is not cut without need.  A piece
// that is a whole (sequence, head) is finished in place; others leave their unnormalised sums and the
// maxima they are relative to in `partial`, which a second kernel joins in the order of the blocks
// (no atomics: results do not vary).  That kernel is placed while the first one runs and does its own
// scan meanwhile.
//
// Inside a block every warp is on its own: it copies KEYS rows of K and V with cp.async into its own
// ring in shared memory (16 bytes a lane, rows past the end zero-filled, so that nothing that an
// unwritten slot holds reaches a product), and multiplies with mma.sync m16n8k16: the 16 rows are
// query heads, which is why tcgen05 with its 64 or 128 rows is not used: the products are a
// sixteenth of what those tiles would pad them to, and the copies, not the products, are the
// time.  Up to 8 query heads fill half of the rows; the other half of the second product's
// rows then carry what rounding P to 16 bits has dropped, so P enters with 22 (f16) or 16 (bf16) bits
// and only the result is rounded.  For 9 and more heads that takes a second product.
//
// 8-bit rows.  Codes become f16 exactly on their way into the products.  The query is scaled by a
// power of two per row to fit f16; a key's scale multiplies its score.  A value's scale is folded into
// the weight as exp2(s_j + log2 v_scale_j - M) with M the running maximum of that sum, so the weights
// that enter the product are at most 1 and the largest of them is, however the scales differ; the
// denominator keeps its own maximum and f32 weights.
#include <type_traits>

#include "cache.cuh"

namespace b200 {
namespace {

using heads::View1;
using heads::View2;
using heads::View3;
using heads::View4;

constexpr int kWarps = 4;
constexpr int kBlock = kWarps * 32;
constexpr int kBlocksPerSm = 2;
constexpr int kJoinThreads = 256;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

struct Problem {
  const void *q;
  int64_t q_batch, q_head;                       // elements
  const uint8_t *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;   // bytes
  const float *k_scale, *v_scale;
  int64_t ks_page, ks_head, ks_slot, vs_page, vs_head, vs_slot;
  const int *table;
  int64_t table_row, table_column;
  const int *lengths;
  int64_t lengths_step;
  void *out;
  int64_t out_batch, out_head;
  float *lse;
  int64_t lse_batch, lse_head;
  float *partial;
  int batch, kv_heads, group, row_tiles, page_size, pages, runs;
  int64_t most_keys;                             // slots that a row of the table names
  float scale_log2e;
  int *status;
};

template <int STORE, int D> struct Shape {
  static constexpr int kBytes = STORE == cache::kNative ? 2 : 1;
  static constexpr int kKeys = STORE == cache::kNative ? 16 : 32;   // key positions of a warp's tile
  static constexpr int kStep = kWarps * kKeys;
  static constexpr int kRowBytes = D * kBytes;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kStages = D == 128 ? 3 : 4;                  // 64 KB of copies in flight on an SM, or more
  static constexpr int kScaleBytes = STORE == cache::kNative ? 0 : 2 * kKeys * 4;
  static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
};
template <int STORE, int D, int ROWS> constexpr int smem_bytes() {
  return Shape<STORE, D>::kRingBytes + ROWS * D * 4 + kWarps * ROWS * 3 * 4;
}
constexpr int partial_floats(int columns) { return columns + 4; }   // sums, m, l, M, unused

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
__device__ __forceinline__ void load_matrix(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void load_matrix_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
template <typename M>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(M) == 2 && !std::is_same<M, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename M> __device__ __forceinline__ uint32_t pack(float low, float high) {
  const M a = Element<M>::narrow(low), b = Element<M>::narrow(high);
  return (uint32_t)*reinterpret_cast<const uint16_t *>(&a) | (uint32_t)*reinterpret_cast<const uint16_t *>(&b) << 16;
}
template <typename M> __device__ __forceinline__ float unpack(uint32_t pair, int i) {
  const uint16_t bits = (uint16_t)(pair >> (16 * i));
  return Element<M>::widen(*reinterpret_cast<const M *>(&bits));
}

// Two 8-bit codes of `word`, at bytes I and J, as f16 (exact).
template <int STORE, int I, int J> __device__ __forceinline__ uint32_t codes(uint32_t word) {
  if constexpr (STORE == cache::kInt8) {
    // 0x6400 + u is 1024 + u in f16; u = code + 128 (the sign bit flipped)
    const uint32_t biased = __byte_perm(word ^ 0x80808080u, 0x64646464u, I | 4 << 4 | J << 8 | 4 << 12);
    const __half2 less = __hsub2(*reinterpret_cast<const __half2 *>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&less);
  } else {
    return cache::f16x2_of_e4m3(__byte_perm(word, 0, I | J << 4));
  }
}

template <int CHUNKS> __device__ __forceinline__ int swizzled(int row, int chunk) {
  // eight neighbouring rows at one chunk fall into eight different groups of four banks
  return chunk ^ (CHUNKS >= 8 ? row & 7 : (row >> 1) & 3);
}

__device__ __forceinline__ int length_of(const Problem &p, int b) {
  const int length = p.lengths[b * p.lengths_step];
  return length <= 0 ? 0 : (int)min((int64_t)length, p.most_keys);
}

// Sum over the block of `v`, and the sum over the threads before this one.
template <int THREADS> __device__ __forceinline__ int64_t block_scan(int64_t v, int64_t &before, int64_t *scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inclusive = v;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, inclusive, offset);
    if (lane >= offset) inclusive += other;
  }
  __syncthreads();   // the scratch may still be read
  if (lane == 31) scratch[warp] = inclusive;
  __syncthreads();
  int64_t total = 0;
  before = inclusive - v;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  return total;
}

struct Place {            // where in the sequence of steps a warp is
  int b, head, step, steps, length;
  int64_t left;
  template <int STEP> __device__ __forceinline__ void advance(const Problem &p) {
    --left;
    if (++step < steps) return;
    step = 0;
    if (++head < p.kv_heads * p.row_tiles) return;
    head = 0;
    if (left <= 0) return;
    do {
      if (++b >= p.batch) {   // only if the lengths change under the kernel
        left = 0;
        return;
      }
      length = length_of(p, b);
    } while (length == 0);
    steps = (length + STEP - 1) / STEP;
  }
};

template <typename T, int STORE, int D, int ROWS>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm)
paged_attention_kernel(const Problem p) {
  using S = Shape<STORE, D>;
  using M = typename std::conditional<STORE == cache::kNative, T, __half>::type;   // type of the products
  constexpr bool kCodes = STORE != cache::kNative;
  constexpr int kHalves = ROWS / 8, kTiles = S::kKeys / 8;
  extern __shared__ __align__(128) unsigned char dynamic_smem[];
  __shared__ int64_t scan_scratch[kWarps];
  __shared__ int64_t start_rest;
  __shared__ int start_b;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;

  // ---- this block's run of steps
  const int head_tiles = p.kv_heads * p.row_tiles;
  int64_t total = 0, before = 0;
  for (int base = 0; base < p.batch; base += kBlock) {
    const int b = base + threadIdx.x;
    const int length = b < p.batch ? length_of(p, b) : 0;
    if (blockIdx.x == 0 && b < p.batch && p.lengths[b * p.lengths_step] > p.most_keys) heads::report_index(p.status, b);
    total += block_scan<kBlock>((length + S::kStep - 1) / S::kStep, before, scan_scratch);
  }
  total *= head_tiles;
  const int64_t runs = min((int64_t)p.runs, total);   // none is empty, which the join relies on
  if (blockIdx.x >= runs) return;
  const int64_t begin = total * blockIdx.x / runs, end = total * (blockIdx.x + 1) / runs;
  int64_t carried = 0;
  for (int base = 0; base < p.batch; base += kBlock) {
    const int b = base + threadIdx.x;
    const int64_t steps = b < p.batch ? (length_of(p, b) + S::kStep - 1) / S::kStep : 0;
    const int64_t sum = block_scan<kBlock>(steps, before, scan_scratch);
    const int64_t first = (carried + before) * head_tiles;
    if (begin >= first && begin < first + steps * head_tiles) {
      start_b = b;
      start_rest = begin - first;
    }
    carried += sum;
    if (carried * head_tiles > begin) break;
  }
  __syncthreads();
  Place load;             // where the next copies are from
  load.b = start_b;
  load.length = length_of(p, load.b);
  load.steps = (load.length + S::kStep - 1) / S::kStep;
  load.head = (int)(start_rest / load.steps);
  load.step = (int)(start_rest - (int64_t)load.head * load.steps);
  load.left = end - begin;
  Place use = load;       // what the next products take

  // ---- copies: lane r looks row r of the tile up; a row's 16-byte pieces go to neighbouring lanes
  unsigned char *ring = dynamic_smem + warp * S::kStages * S::kStageBytes;
  const uint32_t ring_address = shared_address(ring);
  float *merged = reinterpret_cast<float *>(dynamic_smem + S::kRingBytes);
  float *stats = merged + ROWS * D;
  int entry = -1, offset = 0;
  bool inside = false;
  auto look_up = [&]() {
    inside = false;
    if (load.left <= 0) return;
    const int64_t key = (int64_t)(load.step * kWarps + warp) * S::kKeys + lane;
    inside = lane < S::kKeys && key < load.length;
    if (inside) {
      const uint32_t column = (uint32_t)key / (uint32_t)p.page_size;
      offset = (int)((uint32_t)key - column * (uint32_t)p.page_size);
      entry = __ldg(p.table + load.b * p.table_row + column * p.table_column);
    }
  };
  const bool one_layout = p.k_page == p.v_page && p.k_head == p.v_head && p.k_slot == p.v_slot;
  uint32_t masks[S::kStages - 1];     // which rows of the tiles in flight are there, oldest first
  auto issue = [&](int stage) -> uint32_t {
    bool live = inside;
    if (live && (uint32_t)entry >= (uint32_t)p.pages) {   // never read: the position counts as absent
      heads::report_index(p.status, load.b);
      live = false;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, live);
    if (mask == 0) return 0;
    const int kv_head = load.head / p.row_tiles;
    const int64_t page = live ? entry : 0;
    const int64_t k_row = page * p.k_page + kv_head * p.k_head + (live ? offset : 0) * p.k_slot;
    const int64_t v_row = page * p.v_page + kv_head * p.v_head + (live ? offset : 0) * p.v_slot;
    const uint32_t stage_address = ring_address + stage * S::kStageBytes;
    constexpr int kRowsAtOnce = 32 / S::kChunks;
    const int chunk = lane % S::kChunks;
#pragma unroll
    for (int i = 0; i < S::kKeys / kRowsAtOnce; ++i) {
      const int row = i * kRowsAtOnce + lane / S::kChunks;
      const bool row_live = mask >> row & 1;
      const int64_t from = __shfl_sync(0xffffffffu, k_row, row);
      const uint32_t to = stage_address + row * S::kRowBytes + swizzled<S::kChunks>(row, chunk) * 16;
      copy16(to, p.k + from + chunk * 16, row_live);
      const int64_t v_from = one_layout ? from : __shfl_sync(0xffffffffu, v_row, row);
      copy16(to + S::kTileBytes, p.v + v_from + chunk * 16, row_live);
    }
    if constexpr (kCodes) {
      const uint32_t to = stage_address + 2 * S::kTileBytes + lane * 4;
      copy4(to, p.k_scale + (live ? page * p.ks_page + kv_head * p.ks_head + offset * p.ks_slot : 0), live);
      copy4(to + S::kKeys * 4, p.v_scale + (live ? page * p.vs_page + kv_head * p.vs_head + offset * p.vs_slot : 0), live);
    }
    return mask;
  };
  auto produce = [&](int stage) -> uint32_t {
    uint32_t mask = 0;
    if (load.left > 0) {
      mask = issue(stage);
      load.advance<S::kStep>(p);
      look_up();
    }
    copies_commit();
    return mask;
  };

  // ---- the query rows of the current head, as the products' left operand
  uint32_t query[D / 16][2 * kHalves];
  float row_scale[kHalves];
  auto load_query = [&]() {
    const int kv_head = use.head / p.row_tiles, row0 = (use.head - kv_head * p.row_tiles) * ROWS;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = row0 + h * 8 + g;
      const T *source = static_cast<const T *>(p.q) + use.b * p.q_batch + (kv_head * p.group + min(row, p.group - 1)) * p.q_head;
      const bool live = row < p.group;
      if constexpr (!kCodes) {
        row_scale[h] = p.scale_log2e;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {   // columns 16 i + 2 c, + 1 and 16 i + 8 + 2 c, + 1
          query[i][h] = live ? *reinterpret_cast<const uint32_t *>(source + 16 * i + 2 * c) : 0u;
          query[i][kHalves + h] = live ? *reinterpret_cast<const uint32_t *>(source + 16 * i + 8 + 2 * c) : 0u;
        }
      } else {
        uint2 raw[D / 16];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {   // columns 16 i + 4 c .. + 3
          raw[i] = live ? *reinterpret_cast<const uint2 *>(source + 16 * i + 4 * c) : make_uint2(0, 0);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            most = fmaxf(most, fmaxf(fabsf(unpack<T>(raw[i].x, j)), fabsf(unpack<T>(raw[i].y, j))));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the power of two that brings the row's largest entry into [16, 32): f16 then holds all of a bf16's
        // bits down to 2^-28 of that entry
        const int exponent = (int)(__float_as_uint(most) >> 23) - 127;
        const bool scaled = most > 0.0f && most < INFINITY;
        const int shift = scaled ? min(4 - exponent, 120) : 0;
        const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
        row_scale[h] = p.scale_log2e * __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          query[i][h] = pack<__half>(unpack<T>(raw[i].x, 0) * up, unpack<T>(raw[i].x, 1) * up);
          query[i][kHalves + h] = pack<__half>(unpack<T>(raw[i].y, 0) * up, unpack<T>(raw[i].y, 1) * up);
        }
      }
    }
  };

  // ---- running state of a piece
  float sums[D / 8][4], m[kHalves], l[kHalves], weight_max[kHalves];
  int piece_first = use.step;
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[i][j] = 0.0f;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) { m[h] = weight_max[h] = -INFINITY; l[h] = 0.0f; }
    piece_first = use.step;
  };

  auto consume = [&](int stage, uint32_t mask) {
    const uint32_t k_address = ring_address + stage * S::kStageBytes, v_address = k_address + S::kTileBytes;
    const float *k_scales = reinterpret_cast<const float *>(ring + stage * S::kStageBytes + 2 * S::kTileBytes);
    float s[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] = 0.0f;
    const int low_row = lane & 7;
    // scores: four chunks of eight keys at a time
#pragma unroll
    for (int i = 0; i < S::kChunks / 4; ++i) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        uint32_t r[4];
        const int row = 8 * t + low_row;
        load_matrix(r, k_address + row * S::kRowBytes + swizzled<S::kChunks>(row, 4 * i + (lane >> 3)) * 16);
        if constexpr (!kCodes) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t *a = query[2 * i + j];
            multiply<M>(s[t], a[0], kHalves == 2 ? a[1] : 0u, a[kHalves], kHalves == 2 ? a[3] : 0u, r[2 * j], r[2 * j + 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t *a = query[4 * i + j];
            multiply<M>(s[t], a[0], kHalves == 2 ? a[1] : 0u, a[kHalves], kHalves == 2 ? a[3] : 0u,
                        codes<STORE, 0, 1>(r[j]), codes<STORE, 2, 3>(r[j]));
          }
        }
      }
    }
    // weights: thread (g, c) holds keys 8 t + 2 c, + 1 of rows g and, with 16 rows, g + 8
    float log_scale[kTiles][2];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const uint32_t bits = mask >> (8 * t + 2 * c);
      float2 ks = make_float2(1.0f, 1.0f);
      if constexpr (kCodes) {
        ks = *reinterpret_cast<const float2 *>(k_scales + 8 * t + 2 * c);
        const float2 vs = *reinterpret_cast<const float2 *>(k_scales + S::kKeys + 8 * t + 2 * c);
        log_scale[t][0] = __log2f(vs.x);
        log_scale[t][1] = __log2f(vs.y);
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        s[t][2 * h] = bits & 1 ? s[t][2 * h] * (row_scale[h] * ks.x) : -INFINITY;
        s[t][2 * h + 1] = bits & 2 ? s[t][2 * h + 1] * (row_scale[h] * ks.y) : -INFINITY;
      }
    }
    float new_m[kHalves], new_max[kHalves];
    bool grown = false;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      new_m[h] = m[h];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) new_m[h] = fmaxf(new_m[h], fmaxf(s[t][2 * h], s[t][2 * h + 1]));
      new_m[h] = fmaxf(new_m[h], __shfl_xor_sync(0xffffffffu, new_m[h], 1));
      new_m[h] = fmaxf(new_m[h], __shfl_xor_sync(0xffffffffu, new_m[h], 2));
      new_max[h] = new_m[h];
      if constexpr (kCodes) {
        new_max[h] = weight_max[h];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
          new_max[h] = fmaxf(new_max[h], fmaxf(s[t][2 * h] + log_scale[t][0], s[t][2 * h + 1] + log_scale[t][1]));
        new_max[h] = fmaxf(new_max[h], __shfl_xor_sync(0xffffffffu, new_max[h], 1));
        new_max[h] = fmaxf(new_max[h], __shfl_xor_sync(0xffffffffu, new_max[h], 2));
      }
      grown |= new_m[h] > m[h] || new_max[h] > weight_max[h];
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        l[h] *= exp2_fast(m[h] - finite_or_zero(new_m[h]));
        const float shrink = exp2_fast(weight_max[h] - finite_or_zero(new_max[h]));
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          sums[i][2 * h] *= shrink;
          sums[i][2 * h + 1] *= shrink;
          if (kHalves == 1) {   // the other half of the rows belongs to the same heads
            sums[i][2] *= shrink;
            sums[i][3] *= shrink;
          }
        }
        m[h] = new_m[h];
        weight_max[h] = new_max[h];
      }
    }
    uint32_t high[kTiles][kHalves], rest[kTiles][kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const float base = finite_or_zero(m[h]), weight_base = finite_or_zero(weight_max[h]);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        float w0 = exp2_fast(s[t][2 * h] - base), w1 = exp2_fast(s[t][2 * h + 1] - base);
        l[h] += w0 + w1;
        if constexpr (kCodes) {   // log2 of a masked key's zero scale is -infinity: its weight is 0
          w0 = exp2_fast(s[t][2 * h] + log_scale[t][0] - weight_base);
          w1 = exp2_fast(s[t][2 * h + 1] + log_scale[t][1] - weight_base);
        }
        high[t][h] = pack<M>(w0, w1);
        rest[t][h] = pack<M>(w0 - unpack<M>(high[t][h], 0), w1 - unpack<M>(high[t][h], 1));
      }
    }
    // sums += weights . values: two chunks of sixteen keys at a time
#pragma unroll
    for (int b = 0; b < S::kKeys / 16; ++b) {
#pragma unroll
      for (int i = 0; i < S::kChunks / 2; ++i) {
        uint32_t r[4];
        const int row = 16 * b + low_row + (lane & 8);
        load_matrix_transposed(r, v_address + row * S::kRowBytes + swizzled<S::kChunks>(row, 2 * i + (lane >> 4)) * 16);
        const uint32_t *h0 = high[2 * b], *h1 = high[2 * b + 1], *r0 = rest[2 * b], *r1 = rest[2 * b + 1];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (!kCodes) {
            float(&to)[4] = sums[2 * i + j];
            if constexpr (kHalves == 1) {
              multiply<M>(to, h0[0], r0[0], h1[0], r1[0], r[2 * j], r[2 * j + 1]);
            } else {
              multiply<M>(to, h0[0], h0[1], h1[0], h1[1], r[2 * j], r[2 * j + 1]);
              multiply<M>(to, r0[0], r0[1], r1[0], r1[1], r[2 * j], r[2 * j + 1]);
            }
          } else {   // a 16-bit unit holds two neighbouring columns: even and odd ones make a tile each
            const uint32_t even0 = codes<STORE, 0, 2>(r[2 * j]), even1 = codes<STORE, 0, 2>(r[2 * j + 1]);
            const uint32_t odd0 = codes<STORE, 1, 3>(r[2 * j]), odd1 = codes<STORE, 1, 3>(r[2 * j + 1]);
            float(&to_even)[4] = sums[2 * (2 * i + j)];
            float(&to_odd)[4] = sums[2 * (2 * i + j) + 1];
            if constexpr (kHalves == 1) {
              multiply<M>(to_even, h0[0], r0[0], h1[0], r1[0], even0, even1);
              multiply<M>(to_odd, h0[0], r0[0], h1[0], r1[0], odd0, odd1);
            } else {
              multiply<M>(to_even, h0[0], h0[1], h1[0], h1[1], even0, even1);
              multiply<M>(to_odd, h0[0], h0[1], h1[0], h1[1], odd0, odd1);
              multiply<M>(to_even, r0[0], r0[1], r1[0], r1[1], even0, even1);
              multiply<M>(to_odd, r0[0], r0[1], r1[0], r1[1], odd0, odd1);
            }
          }
        }
      }
    }
  };

  // ---- the end of a piece: the warps' states are added up, warp after warp
  auto finish = [&](bool whole) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (c == 0) {
        float *mine = stats + (warp * ROWS + h * 8 + g) * 3;
        mine[0] = m[h];
        mine[1] = l[h];
        mine[2] = weight_max[h];
      }
    }
    __syncthreads();
    auto most = [&](int row, int word) {
      float v = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = fmaxf(v, stats[(w * ROWS + row) * 3 + word]);
      return v;
    };
    float shrink[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) shrink[h] = exp2_fast(weight_max[h] - finite_or_zero(most(h * 8 + g, 2)));
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          float *row = merged + (h * 8 + g) * D;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float(&from)[4] = sums[2 * i + n];
                x[2 * n + j] = (kHalves == 1 ? from[j] + from[2 + j] : from[2 * h + j]) * shrink[h];
              }
            if constexpr (!kCodes) {   // tiles 2 i, 2 i + 1: columns 16 i + 2 c, + 1 and 16 i + 8 + 2 c, + 1
              float2 *to0 = reinterpret_cast<float2 *>(row + 16 * i + 2 * c), *to1 = to0 + 4;
              const float2 old0 = w ? *to0 : make_float2(0.0f, 0.0f), old1 = w ? *to1 : make_float2(0.0f, 0.0f);
              *to0 = make_float2(old0.x + x[0], old0.y + x[1]);
              *to1 = make_float2(old1.x + x[2], old1.y + x[3]);
            } else {                   // even and odd columns of 16 i + 4 c .. + 3
              float4 *to = reinterpret_cast<float4 *>(row + 16 * i + 4 * c);
              const float4 old = w ? *to : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              *to = make_float4(old.x + x[0], old.y + x[2], old.z + x[1], old.w + x[3]);
            }
          }
        }
      }
      __syncthreads();
    }
    const int kv_head = use.head / p.row_tiles, row0 = (use.head - kv_head * p.row_tiles) * ROWS;
    const int rows = min(ROWS, p.group - row0);
    for (int index = threadIdx.x; index < rows * D; index += kBlock) {
      const int row = index / D, column = index % D;
      const float top = most(row, 0), weight_top = most(row, 2);
      float denominator = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        denominator += stats[(w * ROWS + row) * 3 + 1] * exp2_fast(stats[(w * ROWS + row) * 3] - finite_or_zero(top));
      const int head = kv_head * p.group + row0 + row;
      if (whole) {
        const float unit = kCodes ? exp2_fast(finite_or_zero(weight_top) - finite_or_zero(top)) : 1.0f;
        static_cast<T *>(p.out)[use.b * p.out_batch + head * p.out_head + column] =
            Element<T>::narrow(__fdiv_rn(merged[index] * unit, denominator));
        if (column == 0 && p.lse) p.lse[use.b * p.lse_batch + head * p.lse_head] = (finite_or_zero(top) + log2f(denominator)) * kLn2;
      } else {
        // slot 1 if the piece begins its head (only a run's last piece may then be unfinished), else slot 0
        float *to = p.partial + (((int64_t)blockIdx.x * 2 + (piece_first == 0)) * ROWS + row) * partial_floats(D);
        to[column] = merged[index];
        if (column == 0) {
          to[D] = top;
          to[D + 1] = denominator;
          to[D + 2] = weight_top;
        }
      }
    }
    __syncthreads();   // `merged` and `stats` are free again
  };

  // ---- the run
  look_up();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) masks[i] = produce(i);
  load_query();
  reset();
  int stage = 0;
  while (use.left > 0) {
    const int free_stage = stage == 0 ? S::kStages - 1 : stage - 1;
    const uint32_t newest = produce(free_stage);
    copies_wait<S::kStages - 1>();
    __syncwarp();
    if (masks[0]) consume(stage, masks[0]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < S::kStages - 2; ++i) masks[i] = masks[i + 1];
    masks[S::kStages - 2] = newest;
    stage = stage == S::kStages - 1 ? 0 : stage + 1;
    const bool ends = use.step == use.steps - 1;
    if (ends || use.left == 1) {
      finish(ends && piece_first == 0);
      use.advance<S::kStep>(p);
      if (use.left > 0) {
        load_query();
        reset();
      }
    } else {
      use.advance<S::kStep>(p);
    }
  }
  copies_wait<0>();
}

// One block joins the pieces of one query head: the runs that hold its steps are contiguous, the
// first piece lies in its run's slot 1 and the others in slot 0.  Heads that one run held are done.
template <typename T, int D, int ROWS, int STEP>
__global__ void __launch_bounds__(kJoinThreads)
paged_attention_join_kernel(const Problem p) {
  constexpr int kLanes = D / 4;                       // threads of a row of sums, four columns each
  constexpr int kRows = kJoinThreads / kLanes;        // pieces at a time
  __shared__ int64_t scratch[kJoinThreads / 32];
  __shared__ float tops[kJoinThreads / 32][2];
  __shared__ float joined[kRows][D + 4];
  const int b = blockIdx.y, head = blockIdx.x;
  const int kv_head = head / p.group, in_group = head - kv_head * p.group;
  const int tile = in_group / ROWS, row = in_group - tile * ROWS;
  const int head_tiles = p.kv_heads * p.row_tiles;
  int64_t total = 0, first = 0, unused;
  for (int base = 0; base < p.batch; base += kJoinThreads) {
    const int other = base + threadIdx.x;
    const int64_t steps = other < p.batch ? (length_of(p, other) + STEP - 1) / STEP : 0;
    total += block_scan<kJoinThreads>(steps, unused, scratch);
    first += block_scan<kJoinThreads>(other < b ? steps : 0, unused, scratch);
  }
  const int length = length_of(p, b), steps = (length + STEP - 1) / STEP;
  total *= head_tiles;
  first = first * head_tiles + (int64_t)(kv_head * p.row_tiles + tile) * steps;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  T *out = static_cast<T *>(p.out) + b * p.out_batch + head * p.out_head;
  if (steps == 0) {
    if (threadIdx.x < D) out[threadIdx.x] = Element<T>::narrow(0.0f);
    if (threadIdx.x == 0 && p.lse) p.lse[b * p.lse_batch + head * p.lse_head] = -INFINITY;
    return;
  }
  // the run of step s is the largest r with total * r / runs <= s
  const int64_t runs = min((int64_t)p.runs, total);
  const int run0 = (int)(((first + 1) * runs - 1) / total), run1 = (int)(((first + steps) * runs - 1) / total);
  if (run0 == run1) return;
  const int pieces = run1 - run0 + 1;
  auto piece = [&](int i) {
    return p.partial + (((int64_t)(run0 + i) * 2 + (i == 0)) * ROWS + row) * partial_floats(D);
  };
  float top = -INFINITY, weight_top = -INFINITY;
  for (int i = threadIdx.x; i < pieces; i += kJoinThreads) {
    const float *from = piece(i);
    top = fmaxf(top, from[D]);
    weight_top = fmaxf(weight_top, from[D + 2]);
  }
  top = warp_max(top);
  weight_top = warp_max(weight_top);
  if ((threadIdx.x & 31) == 0) {
    tops[threadIdx.x >> 5][0] = top;
    tops[threadIdx.x >> 5][1] = weight_top;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    top = fmaxf(top, tops[w][0]);
    weight_top = fmaxf(weight_top, tops[w][1]);
  }
  top = finite_or_zero(top);
  weight_top = finite_or_zero(weight_top);
  const int lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float denominator = 0.0f;
#pragma unroll 4
  for (int i = part; i < pieces; i += kRows) {
    const float *from = piece(i);
    const float4 x = reinterpret_cast<const float4 *>(from)[lane], state = reinterpret_cast<const float4 *>(from)[D / 4];
    const float shrink = exp2_fast(state.z - weight_top);
    denominator += state.y * exp2_fast(state.x - top);
    sum.x += x.x * shrink;
    sum.y += x.y * shrink;
    sum.z += x.z * shrink;
    sum.w += x.w * shrink;
  }
  *reinterpret_cast<float4 *>(&joined[part][4 * lane]) = sum;
  if (lane == 0) joined[part][D] = denominator;
  __syncthreads();
  if (threadIdx.x >= D) return;
  float value = 0.0f;
  denominator = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    value += joined[i][threadIdx.x];
    denominator += joined[i][D];
  }
  out[threadIdx.x] = Element<T>::narrow(__fdiv_rn(value * exp2_fast(weight_top - top), denominator));
  if (threadIdx.x == 0 && p.lse) p.lse[b * p.lse_batch + head * p.lse_head] = (top + log2f(denominator)) * kLn2;
}

// --------------------------------------------------------------------- host
int rows_of(int64_t group) { return group <= 8 ? 8 : 16; }
int step_of(int store) { return store == B200_I8 || store == B200_E4M3 ? Shape<cache::kInt8, 128>::kStep : Shape<cache::kNative, 128>::kStep; }

// As many runs as blocks are resident, or as there can be steps.
int64_t runs_of(int64_t batch, int64_t kv_heads, int64_t group, int64_t most_keys, int store) {
  const int64_t rows = rows_of(group), tiles = kv_heads * ((group + rows - 1) / rows), step = step_of(store);
  const int64_t each = (most_keys + step - 1) / step, resident = (int64_t)kBlocksPerSm * sm_count();
  if (batch == 0 || tiles == 0 || each == 0) return 1;
  if (batch >= resident || tiles >= resident || each >= resident || batch * tiles >= resident) return resident;
  return batch * tiles * each < resident ? batch * tiles * each : resident;
}

template <typename T, int STORE, int D, int ROWS> int launch(const Problem &p, cudaStream_t stream) {
  const auto kernel = paged_attention_kernel<T, STORE, D, ROWS>;
  const size_t bytes = smem_bytes<STORE, D, ROWS>();
  B200_CUDA_TRY(opt_in_dynamic_smem(kernel, bytes));
  kernel<<<p.runs, kBlock, bytes, stream>>>(p);
  B200_CUDA_TRY(cudaGetLastError());
  // placed while the first kernel still runs; it waits for that kernel's end on the device
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(p.kv_heads * p.group, p.batch);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  B200_CUDA_TRY(cudaLaunchKernelEx(&config, paged_attention_join_kernel<T, D, ROWS, Shape<STORE, D>::kStep>, p));
  return B200_OK;
}
template <typename T, int STORE, int D> int by_rows(const Problem &p, cudaStream_t stream) {
  return p.group <= 8 ? launch<T, STORE, D, 8>(p, stream) : launch<T, STORE, D, 16>(p, stream);
}
template <typename T, int STORE> int by_columns(const Problem &p, int columns, cudaStream_t stream) {
  return columns == 64 ? by_rows<T, STORE, 64>(p, stream) : by_rows<T, STORE, 128>(p, stream);
}
template <typename T> int by_store(const Problem &p, int store, int columns, cudaStream_t stream) {
  if (store == B200_I8) return by_columns<T, cache::kInt8>(p, columns, stream);
  if (store == B200_E4M3) return by_columns<T, cache::kE4m3>(p, columns, stream);
  return by_columns<T, cache::kNative>(p, columns, stream);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_attention_scratch(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t keys,
                                            int32_t store, int64_t *words) {
  if (!words || batch < 0 || heads < 0 || kv_heads < 1 || heads % kv_heads || heads > 65536 || keys < 0 || head_dim < 1 || head_dim > 256)
    return fail(B200_ERR_INVALID_ARGUMENT, "paged_attention_scratch: an extent is out of range");
  const int64_t group = heads / kv_heads;
  *words = runs_of(batch, kv_heads, group ? group : 1, keys, store) * 2 * rows_of(group) * partial_floats((int)head_dim);
  return B200_OK;
}

extern "C" int b200_paged_attention(const int64_t *slots, int64_t count, float scale, int32_t dtype, int32_t store, void *stream) {
  const char *what = "paged_attention";
  heads::Slots from(slots, count);
  const View3 q = from.view3();
  cache::Cache held{};
  held.k = from.view4();
  held.v = from.view4();
  held.k_scale = from.view3();
  held.v_scale = from.view3();
  const View2 table = from.view2();
  const View1 lengths = from.view1();
  const View3 out = from.view3();
  const View2 lse = from.view2();
  const View1 partial = from.view1(), workspace = from.view1();
  if (!from.exact()) return fail(B200_ERR_INVALID_ARGUMENT, "%s: %lld slots do not describe its views", what, (long long)count);
  if (dtype != B200_F16 && dtype != B200_BF16) return fail(B200_ERR_INVALID_ARGUMENT, "%s: queries are f16 or bf16", what);
  const int status = cache::check(what, held, dtype, store, 256);
  if (status != B200_OK) return status;
  const View4 &k = held.k, &v = held.v;
  if (!heads::sane(q) || !heads::sane(out) || !heads::sane(table.d0, table.s0) || !heads::sane(table.d1, table.s1) ||
      !heads::sane(lengths.d0, lengths.s0) || !heads::sane(lse.d0, lse.s0) || !heads::sane(lse.d1, lse.s1))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (k.d3 != 64 && k.d3 != 128)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: head_dim %lld is not 64 or 128", what, (long long)k.d3);
  if (q.d2 != k.d3 || out.d0 != q.d0 || out.d1 != q.d1 || out.d2 != q.d2)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: queries, output and cache differ in shape", what);
  if (k.d1 < 1 || q.d1 < 1 || q.d1 % k.d1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the query heads are not a multiple of the cache's heads", what);
  if (q.d0 > 65535 || q.d1 > 65536)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: more than 65535 sequences or 65536 heads", what);
  if (table.d0 != q.d0 || lengths.d0 != q.d0)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: block table, lengths and queries differ in sequences", what);
  if (lse.data && (lse.d0 != q.d0 || lse.d1 != q.d1)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: lse is (sequences, heads)", what);
  if (!isfinite(scale)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: scale is not a finite number", what);
  if (!workspace.data || workspace.d0 < B200_WORKSPACE_WORDS || workspace.s0 != 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the workspace needs %d contiguous int32 words", what, B200_WORKSPACE_WORDS);
  if (q.d0 == 0) return B200_OK;
  if (k.d2 && table.d1 > (INT32_MAX - 4096) / k.d2)   // key positions and steps are counted in int32
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: a row of the block table names 2^31 positions or more", what);
  const int64_t most_keys = table.d1 * k.d2;
  const int64_t group = q.d1 / k.d1, runs = runs_of(q.d0, k.d1, group, most_keys, store);
  if (!q.data || !out.data || !lengths.data || (table.d1 && !table.data) || !partial.data)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (partial.d0 < runs * 2 * rows_of(group) * partial_floats((int)q.d2) || partial.s0 != 1 || !aligned16(partial.data))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the scratch is too short, not contiguous or not 16-byte aligned", what);
  if (!heads::vector_rows(q, 2) || !heads::vector_rows(out, 2))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  const int size = heads::element_size(store);
  const heads::Span to = heads::span(out, 2);
  if (!heads::distinct(out) || heads::overlap(to, heads::span(q, 2)) || heads::overlap(to, heads::span(k, size)) ||
      heads::overlap(to, heads::span(v, size)))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the output overlaps itself or an input", what);

  Problem p{};
  p.q = q.data; p.q_batch = q.s0; p.q_head = q.s1;
  p.k = static_cast<const uint8_t *>(k.data); p.v = static_cast<const uint8_t *>(v.data);
  p.k_page = k.s0 * size; p.k_head = k.s1 * size; p.k_slot = k.s2 * size;
  p.v_page = v.s0 * size; p.v_head = v.s1 * size; p.v_slot = v.s2 * size;
  p.k_scale = static_cast<const float *>(held.k_scale.data); p.v_scale = static_cast<const float *>(held.v_scale.data);
  p.ks_page = held.k_scale.s0; p.ks_head = held.k_scale.s1; p.ks_slot = held.k_scale.s2;
  p.vs_page = held.v_scale.s0; p.vs_head = held.v_scale.s1; p.vs_slot = held.v_scale.s2;
  p.table = static_cast<const int *>(table.data); p.table_row = table.s0; p.table_column = table.s1;
  p.lengths = static_cast<const int *>(lengths.data); p.lengths_step = lengths.s0;
  p.out = const_cast<void *>(out.data); p.out_batch = out.s0; p.out_head = out.s1;
  p.lse = static_cast<float *>(const_cast<void *>(lse.data)); p.lse_batch = lse.s0; p.lse_head = lse.s1;
  p.partial = static_cast<float *>(const_cast<void *>(partial.data));
  p.batch = (int)q.d0; p.kv_heads = (int)k.d1; p.group = (int)group;
  p.row_tiles = (int)((group + rows_of(group) - 1) / rows_of(group));
  p.page_size = (int)k.d2; p.pages = (int)k.d0; p.runs = (int)runs;
  p.most_keys = most_keys;
  p.scale_log2e = scale * kLog2e;
  p.status = static_cast<int *>(const_cast<void *>(workspace.data));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B200_F16 ? by_store<__half>(p, store, (int)q.d2, s) : by_store<__nv_bfloat16>(p, store, (int)q.d2, s);
}
