// Attention of one new token a sequence over a paged key-value cache in 16 or 8 bits.
//
//     s_j = scale (q . k_j)      out = sum_j e^(s_j) v_j / sum_j e^(s_j)      lse = log sum_j e^(s_j)
//
// The cache is read once and is nearly all that is read, so HBM bounds it: 4 D bytes (16 bits) or
// 2 D + 8 (8 bits) for a key position of a head, against 4 D operations for each of the `group` query
// heads that share it.  What the kernel has to do is keep copies in flight on every SM, whatever
// the lengths are.
//
// Work.  The unit is a step: WARPS * KEYS key positions of one (sequence, key head, tile of query heads).  All
// steps of the call, sequence after sequence, are cut into as many equal runs as there are resident
// blocks (of several heads abreast, see heads_abreast); a block finds its run by a scan of the lengths and crosses
// from one sequence to the next without draining its copies.  A ragged batch therefore loads all SMs alike, a single long
// sequence is spread over all of them, and a short one is not cut without need.  A piece
// that is a whole (sequence, head) is finished in place; others leave their unnormalised sums and the
// maxima they are relative to in `partial`, which a second kernel joins in the order of the blocks
// (no atomics: results do not vary).  Only the borders between runs cut heads, so that kernel has a
// block for each border and four rows, which the run's own note tells what it cuts.  Where no sequence can be
// long, each (sequence, head) is a run, and nothing is joined (see whole_heads).
//
// Inside a block every warp is on its own: it copies KEYS rows of K and V with cp.async into its own
// ring in shared memory (16 bytes a lane, rows past the end zero-filled, so that nothing that an
// unwritten slot holds reaches a product), and multiplies with mma.sync m16n8k16.  Keys (and in the second
// product columns of V) are the 16 rows and query heads the 8 columns, so the group sizes of real
// models fill the products without padding; tcgen05's smallest tiles would pad them 2 to 16 times and
// take the weights through shared memory, to speed up what is not the time.  The weights enter the
// second product as the sum of two halves of 16 bits, so that they count with 16 bits (bf16) or with 22, and with
// 2^-43 of the largest where those are finer (f16: the products of f16 rows and of codes, see kLift); the result is
// rounded once.  Up to four query heads stand in the columns twice: the first four carry
// the weights' first halves and the other four the second ones, in one product instead of two.  Second halves are
// scaled in f16; more heads add them apart for that, which costs 8-bit rows of 8 and 16 query heads 2 to 8 % (32 sequences of
// 4096 keys, 16 heads on each of 8 key heads in e4m3: 73 to 79 us) and 16-bit ones nothing.
//
// Measured (device time; floors at the 6447 GB/s of a copy): one sequence of 131072 keys, 32 query and 8 key heads
// of 128 in bf16: 88.8 us (83.3), of which 85 stream at 6.3 TB/s and 4 join; 64 sequences of 100 to 4096 keys: 88.9
// (82.9); 64 of 1000 to 8192 in e4m3: 103 (94.1); 1024 keys of one sequence: 8.5 us, all latency; 8 of up to 300, 32 heads
// of 64, whole: 7.1.
//
// 8-bit rows.  Codes become f16 exactly on their way into the products.  The query is scaled by a
// power of two per row to fit f16; a key's scale multiplies its score.  A value's scale is folded into
// the weight as exp2((s_j - m) + log2 v_scale_j - w), where m is the running maximum of the scores and w that of the
// rest, so the weights that enter the product are at most 1 and the largest of them is, however the scales differ; the
// denominator keeps f32 weights relative to m.  Scores enter differences only: a score of 2^20 has no room for what
// is added to it.
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
constexpr int kJoinThreads = 512, kJoinAtOnce = 8;
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
  int batch, kv_heads, group, row_tiles, page_size, pages;
  int runs, abreast;                             // blocks = runs * abreast
  int whole;                                     // a run is one (sequence, head tile)
  uint32_t page_magic, page_shift, runs_magic;   // for divisions by page_size and by runs
  double inverse_runs;
  int64_t most_keys;                             // slots that a row of the table names
  float scale_log2e, lift;
  int *status;
};

template <int STORE, int D, int ROWS> struct Shape {
  static constexpr int kBytes = STORE == cache::kNative ? 2 : 1;
  static constexpr int kKeys = STORE == cache::kNative ? 16 : 32;   // key positions of a warp's tile
  static constexpr int kStep = kWarps * kKeys;
  static constexpr int kRowBytes = D * kBytes;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kColumns = ROWS < 8 ? 8 : ROWS;              // of the products; a head's twice if ROWS is 4
  static constexpr int kBlocksPerSm = ROWS <= 8 ? 3 : 2;            // 168 or 255 registers
  static constexpr int kStages = (ROWS <= 8 ? 2 : 3) * (128 / D);   // about 200 KB of an SM's shared memory
  static constexpr int kScaleBytes = STORE == cache::kNative ? 0 : 2 * kKeys * 4;
  static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kSmemBytes = kRingBytes + kWarps * kColumns * 16 + ROWS * 4;
  static_assert(kColumns * D * 4 <= kStageBytes, "a warp's sums fit the stage that it has just used");
};
// Weights of the products, relative to the running maximum, are 2^lift times what they stand for, and their second halves
// kRest times: f16 has room up to 2^15 above (the maximum lags by up to 2^8) and none below 2^-24.  Second halves then
// keep what is above 2^-36, and a weight is off by at most 2^-43 of the largest, or 2^-23 of itself.  Without,
// the ends of a softmax were lost behind a key that holds nearly all of it: by 23 % if they lie 2^26 below.
// bf16 has no end there but one above: its largest numbers times a weight of more than 1 are infinite, so its weights stand
// lower by the 2^8 that the maximum may lag.
template <typename M> constexpr bool kHalf = std::is_same<M, __half>::value;
template <typename M> constexpr float kLift = kHalf<M> ? 7.0f : -8.0f;
template <typename M> constexpr float kRest = kHalf<M> ? 2048.0f : 1.0f;
constexpr int partial_floats(int columns) { return columns + 4; }   // sums, m, l, w, unused

// What a run begins with, for the kernel that joins: (sequence, head tile) and how many of its steps lie
// before the run; and what a run holds.
struct Border {
  int64_t each;
  int rest, b, head, step, steps, unused;
};
static_assert(sizeof(Border) == 32, "two vectors");

// Good to 2^-22 of the result: a score of 4 in f32 is no better.  The logarithm of a value's scale (__log2f) is off by two
// units of its last place, 2^-20 for scales of 2^-8, and a weight by as much of itself.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ uint32_t transposed(uint32_t pair) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(pair));
  return r;
}
__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// The four 8-bit codes of a word as f16 (exact): bytes 0, 1 and 2, 3, or with EVEN_ODD bytes 0, 2 and 1, 3.
template <int STORE, bool EVEN_ODD> __device__ __forceinline__ void widen(uint32_t word, uint32_t &first, uint32_t &second) {
  if constexpr (STORE == cache::kInt8) {
    // 0x6400 + u is 1024 + u in f16; u = code + 128 (the sign bit flipped)
    const uint32_t biased = word ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    const uint32_t low = __byte_perm(biased, 0x64646464u, EVEN_ODD ? 0x4240 : 0x4140);
    const uint32_t high = __byte_perm(biased, 0x64646464u, EVEN_ODD ? 0x4341 : 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2 *>(&low), bias), b = __hsub2(*reinterpret_cast<const __half2 *>(&high), bias);
    first = *reinterpret_cast<const uint32_t *>(&a);
    second = *reinterpret_cast<const uint32_t *>(&b);
  } else {
    const uint32_t ordered = EVEN_ODD ? __byte_perm(word, 0, 0x3120) : word;
    asm("{\n\t.reg .b16 low, high;\n\t"
        "mov.b32 {low, high}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, low;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, high;\n\t}"
        : "=r"(first), "=r"(second) : "r"(ordered));
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

// The first step of a run: floor(total * run / runs) for total = each * runs + rest, by parts that need no
// 64-bit division: rest * run is below 2^18, where the rounded-up reciprocal is exact.
__device__ __forceinline__ int64_t run_begin(const Problem &p, int64_t each, int rest, int run) {
  return each * run + __umulhi((uint32_t)(rest * run), p.runs_magic);
}

struct Place {            // where in the sequence of steps a warp is
  int b, head, step, steps, length;
  int64_t left;
  template <int STEP> __device__ __forceinline__ void advance(const Problem &p) {
    --left;
    if (++step < steps) return;
    step = 0;
    head += p.abreast;
    if (head < p.kv_heads * p.row_tiles) return;
    head = head % p.abreast;
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

// Infinities among the values.  A weight is positive however far below the others it lies, so an infinite value gives
// that infinity; two of both signs give NaN, and so does one under a score of -infinity (0 times it).  The products
// cannot be trusted with them: a weight enters as two numbers that may be 0 or of both signs.  They turn out NaN then,
// and the block goes through the piece's rows again: its lanes add up what is not finite in eight columns of every 8th
// or 16th row each, 0 if nothing is (64 sequences of up to 4096 keys with one such value 175 us instead of 86; calls without
// any cost nothing).  An infinite score needs an infinity (or NaN) in its key or query, and one of
// +infinity makes the denominator NaN, so such a row under an infinite value leaves NaN in any case.
__device__ __forceinline__ bool special(uint32_t pair, uint32_t exponent) {   // exponent: all its bits, of both halves
  return (pair & exponent & 0xffffu) == (exponent & 0xffffu) || (pair & exponent & 0xffff0000u) == (exponent & 0xffff0000u);
}
__device__ __forceinline__ bool special(const uint4 &x, uint32_t exponent) {
  return special(x.x, exponent) || special(x.y, exponent) || special(x.z, exponent) || special(x.w, exponent);
}
template <int VECTORS> __device__ __forceinline__ bool special_row(const void *row, uint32_t exponent) {
  bool found = false;
#pragma unroll 1
  for (int i = 0; i < VECTORS; ++i) found |= special(static_cast<const uint4 *>(row)[i], exponent);
  return found;
}
template <typename T> constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;

// Of keys [begin, end) of a head, as many at a time as the block has rows of lanes; `to`: the warp's, (rows of lanes, D).
template <typename T, int D>
__device__ __forceinline__ void special_values(const Problem &p, int b, int kv_head, int begin, int end, float *to) {
  constexpr int kVectors = D * 2 / 16, kRows = 32 / kVectors, kAtOnce = 4, kStride = kWarps * kRows;
  const int lane = threadIdx.x & 31, vector = lane % kVectors, first = (threadIdx.x >> 5) * kRows + lane / kVectors;
  float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int64_t key0 = begin + first; key0 < end; key0 += kAtOnce * kStride) {
    int entry[kAtOnce], offset[kAtOnce];
    uint4 raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int key = (int)min(key0 + i * kStride, (int64_t)end - 1), column = key / p.page_size;
      entry[i] = key0 + i * kStride < end ? p.table[b * p.table_row + column * p.table_column] : -1;
      offset[i] = key - column * p.page_size;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if ((uint32_t)entry[i] < (uint32_t)p.pages)
        raw[i] = *reinterpret_cast<const uint4 *>(p.v + entry[i] * p.v_page + kv_head * p.v_head + offset[i] * p.v_slot + vector * 16);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (!special(raw[i], kExponent<T>)) continue;
      const bool no_weight = special_row<kVectors>(p.k + entry[i] * p.k_page + kv_head * p.k_head + offset[i] * p.k_slot, kExponent<T>);
      const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float value = unpack<T>(words[j / 2], j % 2);
        if (!(fabsf(value) < INFINITY)) sum[j] += no_weight ? NAN : value;
      }
    }
  }
  float4 *mine = reinterpret_cast<float4 *>(to + (lane / kVectors) * D + vector * 8);
  mine[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
  mine[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
}
__device__ __forceinline__ bool any_nan(const float4 &x) { return isnan(x.x) || isnan(x.y) || isnan(x.z) || isnan(x.w); }
// sums, with what is not finite in the place of NaN.
__device__ __forceinline__ float4 replaced(const float4 &sum, const float4 &special) {
  return make_float4(special.x != 0.0f ? special.x : sum.x, special.y != 0.0f ? special.y : sum.y, special.z != 0.0f ? special.z : sum.z,
                     special.w != 0.0f ? special.w : sum.w);
}

template <typename T, int STORE, int D, int ROWS>
__global__ void __launch_bounds__(kBlock, (Shape<STORE, D, ROWS>::kBlocksPerSm))
paged_attention_kernel(const Problem p) {
  using S = Shape<STORE, D, ROWS>;
  using M = typename std::conditional<STORE == cache::kNative, T, __half>::type;   // type of the products
  constexpr bool kCodes = STORE != cache::kNative;
  constexpr int kHeads = S::kColumns / 8, kTiles = S::kKeys / 16;   // tiles of 8 columns (query heads) and of 16 keys
  constexpr bool kTwice = ROWS == 4;
  extern __shared__ __align__(128) unsigned char dynamic_smem[];
  __shared__ int64_t scan_scratch[kWarps];
  __shared__ int64_t start_rest;
  __shared__ int start_b;
  heads::await_stream();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;

  // ---- this block's run of steps, which it goes through for one of every `abreast` heads
  const int head_tiles = p.kv_heads * p.row_tiles / p.abreast;
  const int run = blockIdx.x / p.abreast, lane_head = blockIdx.x - run * p.abreast;
  // sequences that have not begun, and those of a table that names no slot: all that they hold is absent
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const bool begun = p.lengths[b * p.lengths_step] > 0;
    if (begun && p.most_keys > 0) continue;
    T *out = static_cast<T *>(p.out) + b * p.out_batch;
    for (int index = threadIdx.x; index < p.kv_heads * p.group * D; index += kBlock)
      out[(index / D) * p.out_head + index % D] = Element<T>::narrow(begun ? NAN : 0.0f);
    for (int head = threadIdx.x; p.lse && head < p.kv_heads * p.group; head += kBlock)
      p.lse[b * p.lse_batch + head * p.lse_head] = -INFINITY;
  }
  Place load;             // where the next copies are from
  if (p.whole) {
    load.b = blockIdx.x / head_tiles;
    load.head = blockIdx.x - load.b * head_tiles;
    const int given = p.lengths[load.b * p.lengths_step];
    if (given > p.most_keys && load.head == 0 && threadIdx.x == 0) heads::report_index(p.status, load.b);
    load.length = length_of(p, load.b);
    if (load.length == 0) return;
    load.left = load.steps = (load.length + S::kStep - 1) / S::kStep;
    load.step = 0;
  } else {
    int64_t total = 0, before = 0, steps_here = 0;
    for (int base = 0; base < p.batch; base += kBlock) {
      const int b = base + threadIdx.x;
      const int given = b < p.batch ? p.lengths[b * p.lengths_step] : 0;
      const int length = given <= 0 ? 0 : (int)min((int64_t)given, p.most_keys);
      if (blockIdx.x == 0 && given > p.most_keys) heads::report_index(p.status, b);
      steps_here = (length + S::kStep - 1) / S::kStep;
      total += block_scan<kBlock>(steps_here, before, scan_scratch);
    }
    total *= head_tiles;
    // runs of each or each + 1 steps; none is empty, which the join relies on
    int64_t each = 1;
    int rest = 0;
    if (total >= p.runs) {
      each = (int64_t)((double)total * p.inverse_runs);
      rest = (int)(total - each * p.runs);
      if (rest < 0) { --each; rest += p.runs; }
      if (rest >= p.runs) { ++each; rest -= p.runs; }
    }
    Border *border = reinterpret_cast<Border *>(p.partial + (int64_t)gridDim.x * 2 * ROWS * partial_floats(D)) + blockIdx.x;
    if (run >= min((int64_t)p.runs, total)) {
      if (threadIdx.x == 0) border->step = 0;
      return;
    }
    const int64_t begin = run_begin(p, each, rest, run), end = run_begin(p, each, rest, run + 1);
    int64_t carried = 0;
    for (int base = 0; base < p.batch; base += kBlock) {
      const int b = base + threadIdx.x;
      int64_t sum = total;
      if (p.batch > kBlock) {   // else the scan above stands
        steps_here = b < p.batch ? (length_of(p, b) + S::kStep - 1) / S::kStep : 0;
        sum = block_scan<kBlock>(steps_here, before, scan_scratch) * head_tiles;
      }
      const int64_t first = carried + before * head_tiles;
      if (begin >= first && begin < first + steps_here * head_tiles) {
        start_b = b;
        start_rest = begin - first;
      }
      carried += sum;
      if (carried > begin) break;
    }
    __syncthreads();
    load.b = start_b;
    load.length = length_of(p, load.b);
    load.steps = (load.length + S::kStep - 1) / S::kStep;
    load.head = start_rest >> 32 ? (int)(start_rest / load.steps) : (int)((uint32_t)start_rest / (uint32_t)load.steps);
    load.step = (int)(start_rest - (int64_t)load.head * load.steps);
    load.head = load.head * p.abreast + lane_head;
    load.left = end - begin;
    if (threadIdx.x == 0) *border = Border{each, rest, load.b, load.head, load.step, load.steps, 0};
  }
  Place use = load;       // what the next products take

  // ---- copies: lane r looks row r of the tile up; a row's 16-byte pieces go to neighbouring lanes
  unsigned char *ring = dynamic_smem + warp * S::kStages * S::kStageBytes;
  const uint32_t ring_address = shared_address(ring);
  float4 *stats = reinterpret_cast<float4 *>(dynamic_smem + S::kRingBytes);   // m, l, above of the warps' rows
  float *units = reinterpret_cast<float *>(stats + kWarps * S::kColumns);
  int entry = -1, offset = 0;
  bool inside = false;
  auto look_up = [&]() {
    inside = false;
    if (load.left <= 0) return;
    const int64_t key = (int64_t)(load.step * kWarps + warp) * S::kKeys + lane;
    inside = lane < S::kKeys && key < load.length;
    if (inside) {
      // key / page_size: key is below 2^31, so the sum does not carry
      const uint32_t column = (__umulhi((uint32_t)key, p.page_magic) + (uint32_t)key) >> p.page_shift;
      offset = (int)((uint32_t)key - column * (uint32_t)p.page_size);
      entry = __ldg(p.table + load.b * p.table_row + column * p.table_column);
    }
  };
  const bool one_layout = p.k_page == p.v_page && p.k_head == p.v_head && p.k_slot == p.v_slot;
  const bool whole_pages = p.page_size % 16 == 0;
  constexpr int kRowsAtOnce = 32 / S::kChunks;
  constexpr uint32_t kFull = S::kKeys == 32 ? 0xffffffffu : (1u << S::kKeys % 32) - 1;
  const int chunk = lane % S::kChunks;
  const int64_t k_lane = (lane / S::kChunks) * p.k_slot + chunk * 16, v_lane = (lane / S::kChunks) * p.v_slot + chunk * 16;
  uint32_t masks[S::kStages - 1];     // which rows of the tiles in flight are there, oldest first
  auto issue = [&](int stage) -> uint32_t {
    bool live = inside;
    if (live && (uint32_t)entry >= (uint32_t)p.pages) {   // never read: the position counts as absent
      heads::report_index(p.status, load.b);
      live = false;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, live);
    if (mask == 0) return 0;
    const int kv_head = p.row_tiles == 1 ? load.head : load.head / p.row_tiles;
    const int64_t page = live ? entry : 0;
    const int64_t k_row = page * p.k_page + kv_head * p.k_head + (live ? offset : 0) * p.k_slot;
    const int64_t v_row = one_layout ? k_row : page * p.v_page + kv_head * p.v_head + (live ? offset : 0) * p.v_slot;
    const uint32_t stage_address = ring_address + stage * S::kStageBytes;
    if (whole_pages && mask == kFull) {
      // 16 rows at a time lie one slot apart: one exchange for them
#pragma unroll
      for (int t = 0; t < S::kKeys / 16; ++t) {
        const uint8_t *k = p.k + __shfl_sync(0xffffffffu, k_row, 16 * t) + k_lane;
        const uint8_t *v = p.v + __shfl_sync(0xffffffffu, v_row, 16 * t) + v_lane;
#pragma unroll
        for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
          const int row = 16 * t + i * kRowsAtOnce + lane / S::kChunks;
          const uint32_t to = stage_address + row * S::kRowBytes + swizzled<S::kChunks>(row, chunk) * 16;
          copy16(to, k);
          copy16(to + S::kTileBytes, v);
          k += kRowsAtOnce * p.k_slot;
          v += kRowsAtOnce * p.v_slot;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::kKeys / kRowsAtOnce; ++i) {
        const int row = i * kRowsAtOnce + lane / S::kChunks;
        const bool row_live = mask >> row & 1;
        const uint32_t to = stage_address + row * S::kRowBytes + swizzled<S::kChunks>(row, chunk) * 16;
        copy16(to, p.k + __shfl_sync(0xffffffffu, k_row, row) + chunk * 16, row_live);
        copy16(to + S::kTileBytes, p.v + __shfl_sync(0xffffffffu, v_row, row) + chunk * 16, row_live);
      }
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

  // ---- the query heads of the current tile, as the first product's right operand: thread (g, c) holds
  // head g's columns 16 i + 2 c, + 1 and 16 i + 8 + 2 c, + 1 (of codes: 16 i + 4 c .. + 3)
  uint2 query[D / 16][kHeads];
  float head_scale[kHeads][2];        // of heads 2 c, 2 c + 1, whose scores the thread will hold
  auto fetch_query = [&](const Place &at) {
    const int kv_head = at.head / p.row_tiles, row0 = (at.head - kv_head * p.row_tiles) * ROWS;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int row = row0 + (kTwice ? g & 3 : h * 8 + g);
      const T *source = static_cast<const T *>(p.q) + at.b * p.q_batch + (kv_head * p.group + min(row, p.group - 1)) * p.q_head;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        query[i][h] = make_uint2(0, 0);
        if (row >= p.group) continue;
        if constexpr (kCodes) {
          query[i][h] = *reinterpret_cast<const uint2 *>(source + 16 * i + 4 * c);
        } else {
          query[i][h].x = *reinterpret_cast<const uint32_t *>(source + 16 * i + 2 * c);
          query[i][h].y = *reinterpret_cast<const uint32_t *>(source + 16 * i + 8 + 2 * c);
        }
      }
    }
  };
  auto scale_query = [&]() {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      head_scale[h][0] = head_scale[h][1] = p.scale_log2e;
      if constexpr (kCodes) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            most = fmaxf(most, fmaxf(fabsf(unpack<T>(query[i][h].x, j)), fabsf(unpack<T>(query[i][h].y, j))));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the power of two that brings the row's largest entry into [16, 32): f16 then holds all of a bf16's
        // bits down to 2^-28 of that entry
        const int exponent = (int)(__float_as_uint(most) >> 23) - 127;
        const bool scaled = most > 0.0f && most < INFINITY;
        const int shift = scaled ? min(4 - exponent, 120) : 0;
        const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
        const float down = p.scale_log2e * __uint_as_float((uint32_t)(127 - shift) << 23);
        head_scale[h][0] = __shfl_sync(0xffffffffu, down, 8 * c);
        head_scale[h][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint2 raw = query[i][h];
          query[i][h] = make_uint2(pack<__half>(unpack<T>(raw.x, 0) * up, unpack<T>(raw.x, 1) * up),
                                   pack<__half>(unpack<T>(raw.y, 0) * up, unpack<T>(raw.y, 1) * up));
        }
      }
    }
  };

  // ---- running state of a piece; sums: columns (of V) x heads
  float sums[D / 16][kHeads][4], m[kHeads][2], l[kHeads][2], above[kHeads][2];   // above: w, 0 without codes
  int piece_first = use.step;
  auto reset = [&]() {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[i][h][j] = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) { m[h][j] = -INFINITY; above[h][j] = kCodes ? -INFINITY : 0.0f; l[h][j] = 0.0f; }
    }
    piece_first = use.step;
  };

  auto consume = [&](int stage, uint32_t mask) {
    const uint32_t k_address = ring_address + stage * S::kStageBytes, v_address = k_address + S::kTileBytes;
    const float *scales = reinterpret_cast<const float *>(ring + stage * S::kStageBytes + 2 * S::kTileBytes);
    float s[kTiles][kHeads][4];       // scores: keys 16 t + g and + 8, heads 2 c and 2 c + 1
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][h][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kChunks / 2; ++i) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        uint32_t r[4];                // two chunks of keys 16 t .. + 7 and + 8 .. + 15
        const int row = 16 * t + (lane & 15);
        load_matrix(r, k_address + row * S::kRowBytes + swizzled<S::kChunks>(row, 2 * i + (lane >> 4)) * 16);
        if constexpr (!kCodes) {
#pragma unroll
          for (int h = 0; h < kHeads; ++h) multiply<M>(s[t][h], r[0], r[1], r[2], r[3], query[i][h].x, query[i][h].y);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t a0, a1, a2, a3;
            widen<STORE, false>(r[2 * j], a0, a2);
            widen<STORE, false>(r[2 * j + 1], a1, a3);
#pragma unroll
            for (int h = 0; h < kHeads; ++h) multiply<M>(s[t][h], a0, a1, a2, a3, query[2 * i + j][h].x, query[2 * i + j][h].y);
          }
        }
      }
    }
    float log_scale[kTiles][2];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int key = 16 * t + 8 * k + g;
        float key_scale = 1.0f;
        if constexpr (kCodes) {
          key_scale = scales[key];
          log_scale[t][k] = __log2f(scales[S::kKeys + key]);
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) s[t][h][2 * k + j] *= head_scale[h][j] * key_scale;
      }
    if (mask != kFull) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (!(mask >> (16 * t + 8 * k + g) & 1))
#pragma unroll
            for (int h = 0; h < kHeads; ++h) s[t][h][2 * k] = s[t][h][2 * k + 1] = -INFINITY;
    }
    // The bases m and above move only when a score passes them by more than 8 (log2 units): until then
    // weights reach 2^8 times what they stand for at the most, which kLift leaves room for.
    bool grown = false;
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const float d[2] = {s[t][h][j] - m[h][j], s[t][h][2 + j] - m[h][j]};
          grown |= fmaxf(d[0], d[1]) > 8.0f;
          if constexpr (kCodes) grown |= fmaxf(d[0] + log_scale[t][0], d[1] + log_scale[t][1]) > above[h][j] + 8.0f;
        }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float shrink[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = m[h][j];
#pragma unroll
          for (int t = 0; t < kTiles; ++t) top = fmaxf(top, fmaxf(s[t][h][j], s[t][h][2 + j]));
#pragma unroll
          for (int other = 4; other < 32; other <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, other));
          const float base = finite_or_zero(top), moved = m[h][j] - base;
          l[h][j] *= exp2_fast(moved);
          m[h][j] = top;
          if constexpr (kCodes) {
            const float old = above[h][j] + moved;
            float w = old;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              w = fmaxf(w, fmaxf(s[t][h][j] - base + log_scale[t][0], s[t][h][2 + j] - base + log_scale[t][1]));
#pragma unroll
            for (int other = 4; other < 32; other <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, other));
            shrink[j] = exp2_fast(old - finite_or_zero(w));
            above[h][j] = w;
          } else {
            shrink[j] = exp2_fast(moved);
          }
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sums[i][h][j] *= shrink[j & 1];
      }
    }
    uint32_t high[kTiles][kHeads][2], rest[kTiles][kHeads][2];   // head g, keys 16 t + 2 c, + 1 and + 8, + 9
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const float base[2] = {finite_or_zero(m[h][0]), finite_or_zero(m[h][1])};
      const float lift[2] = {kLift<M> - finite_or_zero(above[h][0]), kLift<M> - finite_or_zero(above[h][1])};
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float w[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float d = s[t][h][2 * k + j] - base[j];
            w[j] = exp2_fast(d + kLift<M>);
            l[h][j] += w[j];
            // log2 of a masked key's zero scale is -infinity: its weight is 0
            if constexpr (kCodes) w[j] = exp2_fast(d + (log_scale[t][k] + lift[j]));
          }
          const uint32_t pair = pack<M>(w[0], w[1]), left = pack<M>((w[0] - unpack<M>(pair, 0)) * kRest<M>, (w[1] - unpack<M>(pair, 1)) * kRest<M>);
          high[t][h][k] = transposed(kTwice && c >= 2 ? left : pair);
          if constexpr (!kTwice) rest[t][h][k] = transposed(left);
        }
    }
    // sums += values (transposed) . weights
    auto add_rest = [](float (&to)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
      if constexpr (kRest<M> == 1.0f) {
        multiply<M>(to, a0, a1, a2, a3, b[0], b[1]);
      } else {
        float apart[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        multiply<M>(apart, a0, a1, a2, a3, b[0], b[1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = fmaf(apart[j], 1.0f / kRest<M>, to[j]);
      }
    };
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int i = 0; i < S::kChunks / 2; ++i) {
        uint32_t r[4];                // two chunks of keys 16 t .. + 7, the same of keys + 8 .. + 15
        const int row = 16 * t + (lane & 7) + (lane >> 4) * 8;
        load_matrix_transposed(r, v_address + row * S::kRowBytes + swizzled<S::kChunks>(row, 2 * i + (lane >> 3 & 1)) * 16);
        if constexpr (!kCodes) {
#pragma unroll
          for (int h = 0; h < kHeads; ++h) multiply<M>(sums[i][h], r[0], r[1], r[2], r[3], high[t][h][0], high[t][h][1]);
          if constexpr (!kTwice) {
#pragma unroll
            for (int h = 0; h < kHeads; ++h) add_rest(sums[i][h], r[0], r[1], r[2], r[3], rest[t][h]);
          }
        } else {                      // a 16-bit unit holds two neighbouring columns: even ones are rows 0 .. 7, odd ones 8 .. 15
          uint32_t v[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            widen<STORE, true>(r[j], v[j][0], v[j][1]);
            widen<STORE, true>(r[2 + j], v[j][2], v[j][3]);
          }
#pragma unroll
          for (int h = 0; h < kHeads; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              multiply<M>(sums[2 * i + j][h], v[j][0], v[j][1], v[j][2], v[j][3], high[t][h][0], high[t][h][1]);
          if constexpr (!kTwice) {
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
#pragma unroll
              for (int j = 0; j < 2; ++j) add_rest(sums[2 * i + j][h], v[j][0], v[j][1], v[j][2], v[j][3], rest[t][h]);
          }
        }
      }
    }
  };

  // ---- the end of a piece.  The warps exchange their maxima, bring their sums to the common one and
  // leave them in the stage that they used last; the block adds them up, four columns a thread.
  auto finish = [&](const Place &at, bool whole, int stage) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int other = 4; other < 32; other <<= 1) l[h][j] += __shfl_xor_sync(0xffffffffu, l[h][j], other);
        if (g == 0) stats[warp * S::kColumns + h * 8 + 2 * c + j] = make_float4(m[h][j], l[h][j], above[h][j], 0.0f);
      }
    __syncthreads();
    float *mine = reinterpret_cast<float *>(ring + stage * S::kStageBytes);
    // (row, column) of a warp's sums: eight lanes' columns and four lanes' rows all on different banks
    auto spot = [](int row, int column) { return row * D + (column ^ (row >> 1 & 3) * 8); };
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = h * 8 + 2 * c + j;
        float top = -INFINITY, weight_top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[w * S::kColumns + row].x);
        const float base = finite_or_zero(top);
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          weight_top = fmaxf(weight_top, stats[w * S::kColumns + row].z + (stats[w * S::kColumns + row].x - base));
        float shrink = exp2_fast(above[h][j] + (m[h][j] - base) - finite_or_zero(weight_top));
        if (kTwice && c >= 2) shrink *= 1.0f / kRest<M>;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) mine[spot(row, 16 * i + (kCodes ? 2 * g + k : 8 * k + g))] = sums[i][h][2 * k + j] * shrink;
      }
    const int kv_head = at.head / p.row_tiles, row0 = (at.head - kv_head * p.row_tiles) * ROWS;
    const int rows = min(ROWS, p.group - row0), head0 = kv_head * p.group + row0;
    // slot 1 if the piece begins its head (only a run's last piece may then be unfinished), else slot 0
    float *to = p.partial + ((int64_t)blockIdx.x * 2 + (piece_first == 0)) * ROWS * partial_floats(D);
    if (threadIdx.x < rows) {
      const int row = threadIdx.x;
      float4 state[kWarps];
      float top = -INFINITY, weight_top = -INFINITY, denominator = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        state[w] = stats[w * S::kColumns + row];
        top = fmaxf(top, state[w].x);
      }
      const float base = finite_or_zero(top);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        weight_top = fmaxf(weight_top, state[w].z + (state[w].x - base));
        denominator += state[w].y * exp2_fast(state[w].x - base);
      }
      units[row] = __fdiv_rn(kCodes ? exp2_fast(finite_or_zero(weight_top)) : 1.0f, denominator);
      if (whole) {
        if (p.lse) p.lse[at.b * p.lse_batch + (head0 + row) * p.lse_head] = (base - kLift<M> + log2f(denominator)) * kLn2;
      } else {
        *reinterpret_cast<float4 *>(to + row * partial_floats(D) + D) = make_float4(top, denominator, weight_top, 0.0f);
      }
    }
    __syncthreads();
    bool found = false;
    for (int index = threadIdx.x; index < rows * (D / 4); index += kBlock) {
      const int row = index / (D / 4), column = index % (D / 4) * 4;
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float *from = reinterpret_cast<const float *>(dynamic_smem + (w * S::kStages + stage) * S::kStageBytes);
#pragma unroll
        for (int half = 0; half < (kTwice ? 2 : 1); ++half) {
          const float4 x = *reinterpret_cast<const float4 *>(from + spot(row + 4 * half, column));
          sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
        }
      }
      if constexpr (!kCodes) found |= any_nan(sum) && units[row] < INFINITY;   // the denominator is a number above 0
      if (whole) {
        const float unit = units[row];
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at.b * p.out_batch + (head0 + row) * p.out_head + column) =
            make_uint2(pack<T>(sum.x * unit, sum.y * unit), pack<T>(sum.z * unit, sum.w * unit));
      } else {
        *reinterpret_cast<float4 *>(to + row * partial_floats(D) + column) = sum;
      }
    }
    if constexpr (kCodes) {
      __syncthreads();   // the stage, `stats` and `units` are free again
    } else if (__syncthreads_or(found)) {
      special_values<T, D>(p, at.b, kv_head, piece_first * S::kStep, min((at.step + 1) * S::kStep, at.length), mine);
      __syncthreads();
#pragma unroll 1
      for (int index = threadIdx.x; index < rows * D; index += kBlock) {
        const int row = index / D, column = index % D;
        float extra = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
#pragma unroll
          for (int r = 0; r < 32 / S::kChunks; ++r)
            extra += reinterpret_cast<const float *>(dynamic_smem + (w * S::kStages + stage) * S::kStageBytes)[r * D + column];
        if (extra == 0.0f || !(units[row] < INFINITY)) continue;
        if (special_row<D * 2 / 16>(static_cast<const T *>(p.q) + at.b * p.q_batch + (head0 + row) * p.q_head, kExponent<T>)) extra = NAN;
        T *result = static_cast<T *>(p.out) + at.b * p.out_batch + (head0 + row) * p.out_head + column;
        if (!whole) to[row * partial_floats(D) + column] = extra;
        else *result = Element<T>::narrow(extra);
      }
      __syncthreads();
    }
  };

  // ---- the run
  look_up();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) masks[i] = produce(i);
  fetch_query(use);
  scale_query();
  reset();
  int stage = 0;
  while (use.left > 0) {
    const uint32_t newest = produce(stage == 0 ? S::kStages - 1 : stage - 1);
    copies_wait<S::kStages - 1>();
    __syncwarp();
    if (masks[0]) consume(stage, masks[0]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < S::kStages - 2; ++i) masks[i] = masks[i + 1];
    masks[S::kStages - 2] = newest;
    const bool ends = use.step == use.steps - 1;
    if (ends || use.left == 1) {
      const Place done = use;
      use.advance<S::kStep>(p);
      if (use.left > 0) fetch_query(use);   // on its way while the piece is finished
      finish(done, ends && piece_first == 0, stage);
      if (use.left > 0) {
        scale_query();
        reset();
      }
    } else {
      use.advance<S::kStep>(p);
    }
    stage = stage == S::kStages - 1 ? 0 : stage + 1;
  }
  copies_wait<0>();
}

// Block y joins the pieces of the head that border y cuts, if it is the first one that does: the runs that
// hold the head's steps are contiguous, its first piece lies in its run's slot 1 and the others in slot 0.
// Heads that no border cuts are done.  D / 4 threads take a row, four columns each, and a block up to four rows;
// more threads take more pieces of them, eight at a time, with a running maximum of their own.
struct State {
  float4 sum;
  float denominator, top, weight_top;
};
template <int COUNT> __device__ __forceinline__ void add(State &state, const float4 (&x)[COUNT], const float4 (&other)[COUNT]) {
  float top = state.top;
#pragma unroll
  for (int j = 0; j < COUNT; ++j) top = fmaxf(top, other[j].x);
  const float base = finite_or_zero(top), old = state.weight_top + (state.top - base);
  float weight_top = old;
#pragma unroll
  for (int j = 0; j < COUNT; ++j) weight_top = fmaxf(weight_top, other[j].z + (other[j].x - base));
  const float weight_base = finite_or_zero(weight_top), mine = exp2_fast(old - weight_base);
  state.denominator *= exp2_fast(state.top - base);
  state.sum = make_float4(state.sum.x * mine, state.sum.y * mine, state.sum.z * mine, state.sum.w * mine);
#pragma unroll
  for (int j = 0; j < COUNT; ++j) {
    const float shrink = exp2_fast(other[j].z + (other[j].x - base) - weight_base);
    state.denominator += other[j].y * exp2_fast(other[j].x - base);
    state.sum.x += x[j].x * shrink;
    state.sum.y += x[j].y * shrink;
    state.sum.z += x[j].z * shrink;
    state.sum.w += x[j].w * shrink;
  }
  state.top = top;
  state.weight_top = weight_top;
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads)
paged_attention_join_kernel(const Problem p) {
  constexpr int kLanes = D / 4, kMost = kJoinThreads / kLanes, kAtOnce = kJoinAtOnce;
  __shared__ float4 part_sums[kMost][kLanes];
  __shared__ float4 part_states[kMost];
  const int rows = min(p.group, 4), lane = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
  const int parts = blockDim.x / (kLanes * rows), part = slot / rows, row = blockIdx.y * 4 + slot - part * rows;
  const int block = blockIdx.x + p.abreast, run = block / p.abreast;   // blocks of the first run have no border
  const Border *border = reinterpret_cast<const Border *>(p.partial + (int64_t)p.runs * p.abreast * 2 * ROWS * partial_floats(D)) + block;
  // What follows is short on purpose: every block meets it cold, and instructions that come from L2 cost more
  // than what they do.
  heads::await_stream();
  const Border cut = *border;
  if (cut.step == 0) return;
  const int64_t first = run_begin(p, cut.each, cut.rest, run) - cut.step;
  if (run_begin(p, cut.each, cut.rest, run - 1) > first) return;
  // the head's later runs are those that begin before its end: as many as whole runs fit, or some more
  int pieces = 2 + (cut.each < cut.steps ? (cut.steps - cut.step - 1) / ((int)cut.each + 1) : 0);
  while (run_begin(p, cut.each, cut.rest, run - 1 + pieces) < first + cut.steps) ++pieces;
  State state{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f, -INFINITY, -INFINITY};
  const int64_t pitch = (int64_t)p.abreast * 2 * ROWS * partial_floats(D);      // from a run's pieces to the next one's
  const float *origin = p.partial + ((int64_t)(block - p.abreast) * 2 * ROWS + row) * partial_floats(D);
#pragma unroll 1
  for (int i = part; i < pieces; i += kAtOnce * parts) {
    float4 x[kAtOnce], other[kAtOnce];
    const float *from = origin + i * pitch + (i == 0 ? ROWS * partial_floats(D) : 0);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      other[j] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
      if (i + j * parts < pieces) {
        x[j] = reinterpret_cast<const float4 *>(from)[lane];
        other[j] = reinterpret_cast<const float4 *>(from)[D / 4];
      }
      from = origin + (i + (j + 1) * parts) * pitch;
    }
    add(state, x, other);
  }
  if (parts > 1) {
    part_sums[slot][lane] = state.sum;
    if (lane == 0) part_states[slot] = make_float4(state.top, state.denominator, state.weight_top, 0.0f);
    __syncthreads();
    if (part == 0)
#pragma unroll 1
      for (int i = slot + rows; i < parts * rows; i += rows) {
        const float4 x[1] = {part_sums[i][lane]}, other[1] = {part_states[i]};
        add(state, x, other);
      }
  }
  const int kv_head = cut.head / p.row_tiles, in_group = (cut.head - kv_head * p.row_tiles) * ROWS + row;
  const int head = kv_head * p.group + in_group;
  if (part != 0 || row >= ROWS || in_group >= p.group) return;
  if (any_nan(state.sum) && state.denominator > 0.0f) {
    // a piece's infinity times a weight that is 0 in f32: what counts is what the pieces hold that is not finite
    float4 special = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int i = 0; i < pieces; ++i) {
      const float4 x = reinterpret_cast<const float4 *>(origin + i * pitch + (i == 0 ? ROWS * partial_floats(D) : 0))[lane];
      special = make_float4(special.x + (isfinite(x.x) ? 0.0f : x.x), special.y + (isfinite(x.y) ? 0.0f : x.y),
                            special.z + (isfinite(x.z) ? 0.0f : x.z), special.w + (isfinite(x.w) ? 0.0f : x.w));
    }
    state.sum = replaced(state.sum, special);
  }
  // __fdividef and __log2f: 2 units of the last place, in a few instructions that every block meets cold
  const float base = finite_or_zero(state.top), unit = __fdividef(exp2_fast(finite_or_zero(state.weight_top)), state.denominator);
  T *out = static_cast<T *>(p.out) + cut.b * p.out_batch + head * p.out_head + 4 * lane;
  *reinterpret_cast<uint2 *>(out) = make_uint2(pack<T>(state.sum.x * unit, state.sum.y * unit), pack<T>(state.sum.z * unit, state.sum.w * unit));
  if (lane == 0 && p.lse) p.lse[cut.b * p.lse_batch + head * p.lse_head] = (base - p.lift + __log2f(state.denominator)) * kLn2;
}

// --------------------------------------------------------------------- host
int rows_of(int64_t group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }
int step_of(int store) {
  return store == B200_I8 || store == B200_E4M3 ? Shape<cache::kInt8, 128, 8>::kStep : Shape<cache::kNative, 128, 8>::kStep;
}

// Key heads (and tiles of query heads) that go through a run side by side, in neighbouring blocks: they
// want the same pages at the same time, and what lies next to one another in them.  With token-major pages
// that is the scales of 8 heads in 32 bytes, which heads that follow one another each read from HBM again
// (64 sequences of 4096 keys, 8 heads in e4m3: 119.6 us, abreast 98.6).  The largest divisor up to 16 that
// leaves at most 3% of the resident blocks without a run.
int heads_abreast(int64_t head_tiles, int64_t resident) {
  for (int64_t n = 16; n > 1; --n)
    if (head_tiles % n == 0 && resident / n * n * 100 >= resident * 97) return (int)n;
  return 1;
}

// Whether every (sequence, head tile) gets a block of its own, if the longest sequence that the table has room for is
// short.  It saves the scan of the lengths, the pieces and the join; against it stands that one block goes through
// a head's steps alone.  Device time, split / whole, 8 key heads of 128 with 4 query heads on each in bf16:
// 8 sequences of 128 positions 7.5 / 5.1 us, of 256 8.2 / 7.2, of 512 11.1 / 11.1, of 1024 13.4 / 21.4; one of 256 6.9 / 6.9,
// of 512 7.4 / 10.8; 64 of up to 512 20.8 / 18.0, of 1024 30.5 / 28.9.  In int8: 8 of 256 8.6 / 6.8, of 512 9.7 / 9.5; one of
// 512 7.8 / 8.9; 64 of up to 512 19.0 / 17.1.  Heads of 64: one sequence of 256 6.4 / 5.8, of 512 6.6 / 8.7; 32 of up to
// 512 11.1 / 10.0, of 1024 14.9 / 17.6.  Of 64 to 256 sequences of up to 400 and 512, on 1 to 8 key heads of 4 to 24 query heads
// each, in bf16, int8 and e4m3, whole ones take 2 to 32 % less time, with one exception: where 2048 heads of 16 query heads
// share codes, seven to a resident block, equal runs even the end out and gain up to 3 % (256 of up to 512 in e4m3 83 / 86).
bool whole_heads(int64_t heads, int64_t most_keys, int64_t resident) {
  return heads < (1 << 30) && most_keys <= (2 * heads < resident ? 256 : 512);
}

// As many runs as blocks are resident, or as there can be steps; or a run for each (sequence, head tile).
struct Split {
  int64_t runs, abreast;
  bool whole;
};
Split split_of(int64_t batch, int64_t kv_heads, int64_t group, int64_t most_keys, int store) {
  const int64_t rows = rows_of(group), tiles = kv_heads * ((group + rows - 1) / rows), step = step_of(store);
  const int64_t each = (most_keys + step - 1) / step;
  const int64_t resident = (int64_t)(rows <= 8 ? Shape<cache::kNative, 128, 8>::kBlocksPerSm : Shape<cache::kNative, 128, 16>::kBlocksPerSm) * sm_count();
  if (batch == 0 || tiles == 0 || each == 0) return {1, 1, false};
  if (whole_heads(batch * tiles, most_keys, resident)) return {batch * tiles, 1, true};
  const int64_t abreast = heads_abreast(tiles, resident), most = resident / abreast, groups = tiles / abreast;
  if (batch >= most || groups >= most || each >= most || batch * groups >= most) return {most, abreast, false};
  return {batch * groups * each < most ? batch * groups * each : most, abreast, false};
}

// Words of scratch: two unfinished pieces and a border a block, if heads are cut.
int64_t scratch_words(const Split &split, int64_t group, int64_t columns) {
  return split.whole ? 0 : split.runs * split.abreast * (2 * rows_of(group) * partial_floats((int)columns) + (int64_t)(sizeof(Border) / 4));
}

template <typename T, int STORE, int D, int ROWS> int launch(const Problem &p, cudaStream_t stream) {
  const auto kernel = paged_attention_kernel<T, STORE, D, ROWS>;
  const size_t bytes = Shape<STORE, D, ROWS>::kSmemBytes;
  B200_CUDA_TRY(opt_in_dynamic_smem(kernel, bytes));
  B200_CUDA_TRY(heads::launch_early(kernel, p.runs * p.abreast, kBlock, bytes, stream, p));
  if (p.runs == 1 || p.whole) return B200_OK;   // no border
  // four rows a block; threads for all the pieces that a head has if all are alike, eight to a thread, as far
  // as a block goes
  const int rows = p.group < ROWS ? p.group : ROWS, lanes = (rows < 4 ? rows : 4) * D / 4;
  const int64_t heads = (int64_t)p.batch * (p.kv_heads * p.row_tiles / p.abreast), want = (p.runs / heads + 2 + kJoinAtOnce - 1) / kJoinAtOnce;
  const int parts = (int)(want < kJoinThreads / lanes ? want : kJoinThreads / lanes);
  B200_CUDA_TRY(heads::launch_early(paged_attention_join_kernel<T, D, ROWS>, dim3((p.runs - 1) * p.abreast, (rows + 3) / 4), lanes * parts, 0, stream, p));
  return B200_OK;
}
template <typename T, int STORE, int D> int by_rows(const Problem &p, cudaStream_t stream) {
  if (p.group <= 4) return launch<T, STORE, D, 4>(p, stream);
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
  *words = scratch_words(split_of(batch, kv_heads, group ? group : 1, keys, store), group, head_dim);
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
  const int64_t group = q.d1 / k.d1;
  const Split split = split_of(q.d0, k.d1, group, most_keys, store);
  if (!q.data || !out.data || !lengths.data || (table.d1 && !table.data) || (!split.whole && !partial.data))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!split.whole && (partial.d0 < scratch_words(split, group, q.d2) || partial.s0 != 1 || !aligned16(partial.data)))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the scratch is too short, not contiguous or not 16-byte aligned", what);
  if (!heads::aligned4(table.data) || !heads::aligned4(lengths.data) || !heads::aligned4(lse.data) || !heads::aligned4(workspace.data))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: block table, lengths, lse and workspace are 4-byte aligned", what);
  if (!heads::vector_rows(q, 2) || !heads::vector_rows(out, 2))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  const int size = heads::element_size(store);
  const heads::Span to = heads::span(out, 2);
  if (!heads::distinct(out) || heads::overlap(to, heads::span(q, 2)) || heads::overlap(to, heads::span(k, size)) ||
      heads::overlap(to, heads::span(v, size)))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the output overlaps itself or an input", what);
  using heads::footprint;
  const bool codes = size == 1;
  const heads::Footprint written[] = {footprint(out, 2), lse.data ? footprint(lse, 4) : heads::Footprint(),
                                      split.whole ? heads::Footprint() : footprint(partial, 4), footprint(workspace, 4)};
  const heads::Footprint read[] = {footprint(q, 2), footprint(k, size), footprint(v, size),
                                   codes ? footprint(held.k_scale, 4) : heads::Footprint(),
                                   codes ? footprint(held.v_scale, 4) : heads::Footprint(), footprint(table, 4), footprint(lengths, 4)};
  const int64_t lse_extents[] = {lse.d0, lse.d1}, lse_strides[] = {lse.s0, lse.s1};
  if (lse.data && !heads::distinct(2, lse_extents, lse_strides))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the elements of lse overlap one another", what);
  const int met = heads::check_written(what, written, 4, read, 7);
  if (met != B200_OK) return met;

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
  p.page_size = (int)k.d2; p.pages = (int)k.d0;
  p.runs = (int)split.runs; p.abreast = (int)split.abreast; p.whole = split.whole;
  p.inverse_runs = 1.0 / (double)split.runs;
  p.runs_magic = (uint32_t)(((int64_t(1) << 32) + split.runs - 1) / split.runs - (split.runs == 1));
  p.most_keys = most_keys;
  // 2^shift >= page_size; (magic + 2^32) / 2^(32 + shift) is 1 / page_size to within what 31-bit numbers show
  while ((int64_t(1) << p.page_shift) < k.d2) ++p.page_shift;
  if (k.d2) p.page_magic = (uint32_t)(((int64_t(1) << 32) * ((int64_t(1) << p.page_shift) - k.d2)) / k.d2 + 1);
  p.scale_log2e = scale * kLog2e;
  p.lift = store == B200_BF16 ? kLift<__nv_bfloat16> : kLift<__half>;
  p.status = static_cast<int *>(const_cast<void *>(workspace.data));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B200_F16 ? by_store<__half>(p, store, (int)q.d2, s) : by_store<__nv_bfloat16>(p, store, (int)q.d2, s);
}
