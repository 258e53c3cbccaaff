// Paged causal attention of decoded tokens over 4-bit pages (format: packed_cache.cu), bfloat16 queries.
//
// Built for one head size per library: -DPYLON_HEAD_DIM=64 or 128.  Rows of at most 16 packed query rows (tokens x query heads of a KV head); others are
// skipped here.
//
// Mathematics.  A key is k = step (code - zero) per group of channels, so a score is sum over the groups of step (q . code - zero sum(q)): the product
// runs over the codes, and steps and zeros join per key and group, not per element.  Most of the kernel's instructions are the logic ones (64 lanes a cycle and SM)
// that make operands of codes, so the operands are chosen for few of them:
//   A code in the lowest bits of a float16 is the subnormal number code x 2^-24, four bits further up code x 2^-20: masking alone makes operands, one shift and four
//   masks for eight codes.
//   Scores of an attention take them as they are (channels of odd number: the queries are divided by 16, which is exact).  A sum of products of subnormal numbers keeps
//     some 14 bits below the largest query times the largest code, so a score is off by 2^-14 x 15 steps x the largest query in each group, times the scale.
//     That is a bound on the sum over the codes, not on what is left of it: where step zero sum(q) cancels most of that (queries of one sign over keys around
//     zero) it is no share of the score.  Queries are brought to [8, 16) by a power of two per packed row, so that every bfloat16 query has its place.  (Codes as e4m3 bytes would need three instructions, but this device makes float16 numbers of such operands again: 32.3
//     against 27.8 million instructions over 16 x 8,192 keys.)
//   Values, whose sums run over all keys, and keys whose weights are summed (float32 results) go through one half-precision multiply-add on another unit, which
//     makes (code - zero) x 2^-10 of either, exactly and normal.
//   A weight times the step of its values is one float16 number: the reference of the softmax is the running maximum of score + log2(step), not of the score,
//     less LIFT, which keeps that product below 2^15 whatever the values' sizes.  Groups of channels whose steps differ are first brought to one size, by powers of two
//     (up to 2^64) that follow the largest step of each group so far.  A product counts with float16's 11 bits down to 2^-20 of the largest, below that
//     with an absolute error of 2^-31 of it at most: over n keys a channel is off by n x 2^-27 of its group's largest step at most, beside the rounding of weights.
//
// Layout.  Scores are computed transposed: 16 keys are the rows of an m16n8k16 product and the 8 or 16 packed query rows its columns, so no half of a tile
// is empty with up to 8 query heads to a KV head.  Any order of the channels serves a product, so a thread takes 32 (64, 128) contiguous bits of a key's
// codes as its part of every group; weights turn into the second product's operand by movmatrix; a thread's values are the same channels of four keys,
// paired by a byte permutation of their words before the codes are spread.  Each warp takes 32 of a 128-key tile's keys with a softmax of its own and two
// cp.async stages of its own, so no barrier stands in the loop; the four warps meet at the end of a (row, KV head)'s stretch.
//
// Work.  All rows' tiles lie side by side and are cut into equal runs, one per block, whatever the rows' lengths; stretches of a (row, KV head) that are not
// whole leave maximum, sum and weighted values in scratch memory and a second kernel joins them (a kernel of its own, not the last block to arrive: no
// counters, nothing that two graphs could share).
//
// Measured: 64 rows of 8,192 slots, 32 / 8 heads of 128, groups of 128 channels 131 us (4.2 TB/s), groups of 64 and 32 147 and 178 (more steps and zeros to join; bringing
// groups of values to one size is 5 us of either); one row of 131,071 slots 46 us, of 600 slots 8.  What bounds it is latency: issue slots 54 %, the logic unit 49 %, DRAM 41 %
// busy, the 11 or 12 warps an SM that its registers leave room for waiting most for fixed latencies.
//
// The same kernel without values keeps the scores instead (attention_mass: how much weight every key got), and the second kernel turns them into weights.
#include "common.cuh"

#include <cuda_fp16.h>

#ifndef PYLON_HEAD_DIM
#define PYLON_HEAD_DIM 128
#endif

namespace pylon {

constexpr int D = PYLON_HEAD_DIM;
static_assert(D == 64 || D == 128, "the packed decode attention is built for head sizes 64 and 128");
constexpr int TILE = 128, WARPS = 4, WARP_KEYS = 32, STAGES = 2;
constexpr int CODE_BYTES = WARP_KEYS * D / 2;             // of keys or values of a warp's stage
constexpr int ROW_CHUNKS = D / 32;                        // 16-byte pieces of a key's codes
constexpr int SMALL_ROWS = 16;
constexpr float NOTHING = -3.0e38f;                       // a maximum before any score
constexpr float RESCALE_STEP = 8.f;                       // log2: the reference maximum moves when a score is more than this above it
constexpr float LIFT = 6.f;                               // log2: how far below the maximum the reference of weights that meet values is: 2^(6 + 8), times a mantissa, is float16's room
constexpr float SMALLEST = -80.f;                         // log2 of a key's step, at least: a weight of 2^(80 + 14) leaves a sum room
constexpr int MOST_APART = 64;                            // log2: groups are brought together by no more than this

struct PackedParams {
  const __nv_bfloat16* q;
  long long q_stride;
  const unsigned char* k_codes;
  const unsigned short* k_words;
  const unsigned char* v_codes;
  const unsigned short* v_words;
  __nv_bfloat16* out;
  const int* q_start;
  const int* kv_len;
  const int* block_table;
  int table_width, page_size, num_pages, nq, nkv, group, window, rows, blocks;
  int most_packed;         // rows of more packed query rows are not this launch's
  float scale_log2;
  float* part_values;      // [2 * blocks][columns][D]
  float2* part_sums;       // [2 * blocks][columns]: maximum (log2), sum
  int* error;
  // summed weights
  int last, most_slots, score_columns;      // only a row's last `last` tokens; slots from most_slots on are not looked at; columns the scores have room for
  float* scores;           // [rows * nkv][score_columns][most_slots]
  float2* tops;            // [rows * nkv][score_columns]: maximum, 1 / sum, of a (row, KV head) that lies in one block's run
  float* mass;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned smem_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {   // the rest of the 16 bytes becomes zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_half(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8(unsigned a) {
  unsigned b;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(b) : "r"(a));
  return b;
}
// Codes i of both halves of a word as float16 numbers: code x 2^-24 for even i, code x 2^-20 for odd i (y: the word shifted right by 8).
template <int I>
__device__ __forceinline__ unsigned spread(unsigned x, unsigned y) {
  return (I < 2 ? x : y) & (I & 1 ? 0x00F000F0u : 0x000F000Fu);
}
__device__ __forceinline__ __half2 as_half2(unsigned x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ unsigned as_bits(__half2 x) { return *reinterpret_cast<const unsigned*>(&x); }
// The same as (code - zero) x 2^-10; away: -zero x 2^-10.
template <int I>
__device__ __forceinline__ unsigned spread_values(unsigned x, unsigned y, __half2 away) {
  return as_bits(__hfma2(as_half2(spread<I>(x, y)), __float2half2_rn(I & 1 ? 1024.f : 16384.f), away));
}
__device__ __forceinline__ float word_step(unsigned word) { return __uint_as_float((word & 0xFFF0u) << 16); }
__device__ __forceinline__ float word_zero(unsigned word) { return (float)(int)(word & 15u); }

// A row's stretch of tiles.
struct RowPlan {
  int first_token, tokens, length, first_tile, tiles;
  int oldest;   // the first slot that a token sees; the pages of those before it may be gone
};
__device__ __forceinline__ RowPlan row_plan(const PackedParams& p, int row) {
  RowPlan r;
  r.first_token = p.q_start[row];
  r.tokens = p.q_start[row + 1] - r.first_token;
  if (r.tokens > p.last) {   // summed weights: the last ones
    r.first_token += r.tokens - p.last;
    r.tokens = p.last;
  }
  r.length = min(p.kv_len[row], p.most_slots);
  r.first_tile = r.tiles = r.oldest = 0;
  if (r.tokens > 0 && r.tokens <= p.most_packed / p.group && r.length > 0) {
    if (p.window > 0) r.oldest = max(0, r.length - r.tokens - p.window + 1);
    r.first_tile = r.oldest / TILE;
    r.tiles = (r.length + TILE - 1) / TILE - r.first_tile;
  }
  return r;
}

// starts[r]: how many tiles (times KV heads) lie before row r; starts[rows]: all of them.  Called by every thread of the block.
__device__ __forceinline__ void make_plan(const PackedParams& p, int* starts) {
  if (threadIdx.x < 32) {
    int before = 0;
    for (int base = 0; base < p.rows; base += 32) {
      const int row = base + threadIdx.x;
      int upto = row < p.rows ? row_plan(p, row).tiles * p.nkv : 0;
      const int own = upto;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if ((int)threadIdx.x >= offset) upto += other;
      }
      if (row < p.rows) starts[row] = before + upto - own;
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (threadIdx.x == 0) starts[p.rows] = before;
  }
  __syncthreads();
}
__device__ __forceinline__ int plan_row(const int* starts, int rows, int tile) {   // the row that tile number `tile` belongs to
  int low = 0, high = rows - 1;
  while (low < high) {
    const int middle = (low + high + 1) >> 1;
    if (starts[middle] <= tile) low = middle;
    else high = middle - 1;
  }
  return low;
}

// Where a warp's copies are in the block's run.
struct Cursor {
  int tile, row, head, at;      // number of the tile in all, its row and KV head, its place among the row's tiles (from the first visible one)
  int page, place;              // of the warp's first key of the tile: the logical page and the slot in it
  RowPlan plan;
};
__device__ __forceinline__ void cursor_page(Cursor& c, const PackedParams& p, int warp) {
  const int key = (c.plan.first_tile + c.at) * TILE + warp * WARP_KEYS;
  c.page = key / p.page_size;
  c.place = key - c.page * p.page_size;
}
__device__ __forceinline__ void cursor_set(Cursor& c, const PackedParams& p, const int* starts, int tile, int warp) {
  c.tile = tile;
  c.row = plan_row(starts, p.rows, tile);
  c.plan = row_plan(p, c.row);
  const int within = tile - starts[c.row];
  c.head = within / c.plan.tiles;
  c.at = within - c.head * c.plan.tiles;
  cursor_page(c, p, warp);
}
__device__ __forceinline__ void cursor_next(Cursor& c, const PackedParams& p, const int* starts, int total, int warp) {
  ++c.tile;
  if (++c.at < c.plan.tiles) {
    c.place += TILE;
    while (c.place >= p.page_size) {
      c.place -= p.page_size;
      ++c.page;
    }
    return;
  }
  c.at = 0;
  if (++c.head < p.nkv) {
    cursor_page(c, p, warp);
    return;
  }
  if (c.tile < total) cursor_set(c, p, starts, c.tile, warp);
}

// Blocks to an SM, as measured: more of them have fewer registers each and begin more runs.  64 rows of 8,192 slots, 32 / 8 heads, groups of 128 channels of
// heads of 128: attention 131 us with three, 133 with four, 139 with five; its scores alone 130, 112 and 120.  Heads of 64, groups of 64: 93, 93, 102 and
// 107, 94, 98.  16 packed rows, 16 rows of 3,000 slots, groups of 32 channels of 128: 43 with two, 46 with three; scores 34 and 32.
constexpr int blocks_an_sm(int column_tiles, bool mass) {
  const int blocks = D == 64 || mass ? 4 : 3;
  return column_tiles > 1 ? blocks - 1 : blocks;
}

template <int G, bool MASS>
struct Sizes {
  static constexpr int GROUPS = D / G;
  static constexpr int WORD_BYTES = WARP_KEYS * GROUPS * 2;
  static constexpr int SIDES = MASS ? 1 : 2;                                        // keys, and values
  static constexpr int WORDS_AT = SIDES * CODE_BYTES;
  static constexpr int STAGE_BYTES = SIDES * (CODE_BYTES + WORD_BYTES);
  // What a warp makes of its stage's words: keys' (step, step zero) as float pairs (summed weights: the step, and -zero x 2^-10 twice as float16); values'
  // steps as floats, -zero x 2^-10 as float16 by group and key, and log2 of a key's largest step.
  static constexpr int KEY_SCALES = WARP_KEYS * GROUPS * 8, VALUE_STEPS = WARP_KEYS * GROUPS * 4, VALUE_ZEROS = WARP_KEYS * GROUPS * 2, VALUE_SIZES = WARP_KEYS * 4;
  static constexpr int SCALE_BYTES = KEY_SCALES + (MASS ? 0 : VALUE_STEPS + VALUE_ZEROS + VALUE_SIZES);
};
// A stage's codes: piece c of key r.  The exclusive-or spreads what a warp reads at once over the banks: eight keys' 16 bytes (G 32), four keys' 32 (others).
template <int G>
__device__ __forceinline__ unsigned code_offset(int key, int chunk) {
  const int piece = key * ROW_CHUNKS + chunk, line = piece >> 3;
  return (unsigned)(line * 128 + ((piece ^ ((line & 3) << (G == 32 ? 0 : 1))) & 7) * 16);
}

template <int G, bool ALIGNED, bool MASS>
__device__ __forceinline__ void copy_stage(const PackedParams& p, const Cursor& c, unsigned stage, int warp, int lane) {
  using S = Sizes<G, MASS>;
  const int key0 = (c.plan.first_tile + c.at) * TILE + warp * WARP_KEYS;
  const int* table = p.block_table + (size_t)c.row * p.table_width;
  if constexpr (ALIGNED) {   // pages of a multiple of 16 keys: 16 keys lie side by side, half a warp copies each half of the 32
    const int half = lane >> 4, left = lane & 15;
    int logical = c.page, place = c.place + 16 * half, valid = min(16, c.plan.length - key0 - 16 * half);
    if (place >= p.page_size) {
      place -= p.page_size;
      ++logical;
    }
    int page = 0;
    if (valid > 0 && key0 + 16 * half + valid > c.plan.oldest) {
      page = table[logical];
      if (page < 0 || page >= p.num_pages) {
        if (left == 0) atomicExch(p.error, PYLON_ERROR_BAD_PAGE);
        page = 0;
        valid = 0;
      }
    } else {
      valid = 0;
    }
    const size_t row = ((size_t)page * p.nkv + c.head) * p.page_size + (valid > 0 ? place : 0);
    const unsigned char* k = p.k_codes + row * (D / 2) + left * 16;
    const unsigned char* v = p.v_codes + row * (D / 2) + left * 16;
    // Pieces 16 apart: two places in a line's pattern, 512 bytes between every second.
    const unsigned to[2] = {stage + code_offset<G>(16 * half + left / ROW_CHUNKS, left % ROW_CHUNKS),
                            stage + code_offset<G>(16 * half + left / ROW_CHUNKS + 16 / ROW_CHUNKS, left % ROW_CHUNKS)};
    const int first_key = left / ROW_CHUNKS;
#pragma unroll
    for (int i = 0; i < ROW_CHUNKS; ++i) {
      const int bytes = first_key + i * (16 / ROW_CHUNKS) < valid ? 16 : 0;
      copy16(to[i & 1] + (i >> 1) * 512, k + i * 256, bytes);
      if (!MASS) copy16(to[i & 1] + (i >> 1) * 512 + CODE_BYTES, v + i * 256, bytes);
    }
    constexpr int PIECES = S::WORD_BYTES / 32;   // of half the keys' words: 2, 4 or 8
    if (left < S::SIDES * PIECES) {
      const int piece = left % PIECES;
      const bool values = left >= PIECES;
      const int bytes = min(16, max(0, valid * S::GROUPS * 2 - piece * 16));
      copy16(stage + S::WORDS_AT + (values ? S::WORD_BYTES : 0) + half * (S::WORD_BYTES / 2) + piece * 16,
             reinterpret_cast<const char*>((values ? p.v_words : p.k_words) + row * S::GROUPS) + piece * 16, bytes);
    }
  } else {   // any page size: a page for every key, and the words by hand
    const int own = key0 + lane;
    size_t own_row = 0;
    bool there = own < c.plan.length && own >= c.plan.oldest;
    if (there) {
      const int page = table[own / p.page_size];
      if (page < 0 || page >= p.num_pages) {
        atomicExch(p.error, PYLON_ERROR_BAD_PAGE);
        there = false;
      } else {
        own_row = ((size_t)page * p.nkv + c.head) * p.page_size + own % p.page_size;
      }
    }
    const unsigned there_lanes = __ballot_sync(0xffffffffu, there);
#pragma unroll
    for (int i = 0; i < WARP_KEYS * ROW_CHUNKS / 32; ++i) {
      const int piece = lane + 32 * i, key = piece / ROW_CHUNKS, chunk = piece % ROW_CHUNKS;
      const size_t row = __shfl_sync(0xffffffffu, (unsigned long long)own_row, key);
      const unsigned to = stage + code_offset<G>(key, chunk);
      const size_t from = row * (D / 2) + (size_t)chunk * 16;
      const int bytes = (there_lanes >> key) & 1u ? 16 : 0;
      copy16(to, p.k_codes + from, bytes);
      if (!MASS) copy16(to + CODE_BYTES, p.v_codes + from, bytes);
    }
#pragma unroll
    for (int side = 0; side < S::SIDES; ++side)
#pragma unroll
      for (int w = 0; w < S::GROUPS; ++w) {
        const unsigned short word = there ? (side ? p.v_words : p.k_words)[own_row * S::GROUPS + w] : (unsigned short)0;
        asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(stage + S::WORDS_AT + side * S::WORD_BYTES + (lane * S::GROUPS + w) * 2), "h"(word) : "memory");
      }
  }
}

template <int G, int NT, bool ALIGNED, bool MASS>
__global__ void __launch_bounds__(WARPS * 32, blocks_an_sm(NT, MASS)) attention_packed_kernel(const PackedParams p) {
  using S = Sizes<G, MASS>;
  constexpr int GROUPS = S::GROUPS, COLUMNS = NT * 8;
  constexpr int STEPS = G / 16;                 // k16 products to a group
  constexpr int WORDS = G / 32;                 // words of a key's group that a thread has (scores)
  constexpr int MT = G / 16, MINE = G / 8;      // m16 products to a group of values; channels of a group that a thread has
  constexpr int HALVES = WARP_KEYS / 16;
  extern __shared__ __align__(128) unsigned char shared[];
  unsigned char* ring = shared;                                                                  // [WARPS][STAGES][STAGE_BYTES]
  unsigned char* scales = shared + WARPS * STAGES * S::STAGE_BYTES;                                // [WARPS][SCALE_BYTES]
  float2* merge_sums = reinterpret_cast<float2*>(scales + WARPS * S::SCALE_BYTES);                 // [WARPS][COLUMNS]
  float* merge_values = reinterpret_cast<float*>(merge_sums + WARPS * COLUMNS);                    // [WARPS][COLUMNS][D] (none for summed weights)
  int* starts = reinterpret_cast<int*>(merge_values + (MASS ? 0 : WARPS * COLUMNS * D));           // [rows + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  allow_dependents();
  make_plan(p, starts);
  const int total = starts[p.rows], run = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int begin = blockIdx.x * run, end = min(total, begin + run);
  if (begin >= end) return;

  const unsigned my_ring = smem_address(ring) + warp * STAGES * S::STAGE_BYTES;
  float2* key_scales = reinterpret_cast<float2*>(scales + warp * S::SCALE_BYTES);                   // [WARP_KEYS][GROUPS]
  float* value_steps = reinterpret_cast<float*>(scales + warp * S::SCALE_BYTES + S::KEY_SCALES);    // [WARP_KEYS][GROUPS]
  __half* value_zeros = reinterpret_cast<__half*>(value_steps + WARP_KEYS * GROUPS);                // [GROUPS][WARP_KEYS]
  float* value_sizes = reinterpret_cast<float*>(value_zeros + WARP_KEYS * GROUPS);                  // [WARP_KEYS]
  Cursor ahead;
  cursor_set(ahead, p, starts, begin, warp);
  int ahead_stage = 0;
  auto request = [&]() {
    if (ahead.tile < end) {
      copy_stage<G, ALIGNED, MASS>(p, ahead, my_ring + ahead_stage * S::STAGE_BYTES, warp, lane);
      cursor_next(ahead, p, starts, total, warp);
    }
    copy_commit();
    ahead_stage ^= 1;
  };
  request();
  request();

  // Where this thread's codes lie in a stage: keys g and g + 8 of the first 16 (the other 16 follow at a constant distance), and the four keys of its values.
  constexpr int HALF_BYTES = 16 * D / 2;
  unsigned key_at[GROUPS][2], value_at[GROUPS][4];
#pragma unroll
  for (int gr = 0; gr < GROUPS; ++gr) {
    const int key_byte = gr * (G / 2) + t * (G / 8), value_byte = gr * (G / 2) + (G == 32 ? (g >> 1) * 4 : g * (G / 16));
#pragma unroll
    for (int i = 0; i < 2; ++i) key_at[gr][i] = code_offset<G>(g + 8 * i, key_byte >> 4) + (key_byte & 15);
#pragma unroll
    for (int k = 0; k < 4; ++k) value_at[gr][k] = CODE_BYTES + code_offset<G>(2 * t + (k & 1) + 8 * (k >> 1), value_byte >> 4) + (value_byte & 15);
    if constexpr (D == 128) {   // eight keys are four lines: the same place in the pattern
      key_at[gr][1] = key_at[gr][0] + 512;
      value_at[gr][2] = value_at[gr][0] + 512;
      value_at[gr][3] = value_at[gr][1] + 512;
    }
  }

  int tile = begin, stage_index = 0;
  while (tile < end) {   // a (row, KV head)'s stretch in this block's run
    const int row = plan_row(starts, p.rows, tile);
    const RowPlan plan = row_plan(p, row);
    const int head = (tile - starts[row]) / plan.tiles, at = tile - starts[row] - head * plan.tiles, tiles = min(plan.tiles - at, end - tile);
    const bool starts_here = at == 0, ends_here = at + tiles == plan.tiles;
    const int packed = plan.tokens * p.group;

    // The queries: column n of a product is packed row n, that is token n / group and query head n % group.
    unsigned qb[NT][GROUPS * STEPS][2];
    float qsum[NT][GROUPS][2];                         // of this thread's columns of the scores, 2 t and 2 t + 1: minus the queries' sum x 2^-24
    float scale[NT][2];
    int limit[NT][2];                                  // the last slot that a column sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + g;
      const __nv_bfloat16* src = p.q + (size_t)(plan.first_token + n / p.group) * p.q_stride + (size_t)(head * p.group + n % p.group) * D;
      uint4 raw[GROUPS][WORDS];
      float most = 0.f;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          raw[gr][w] = n < packed ? *reinterpret_cast<const uint4*>(src + gr * G + (t * WORDS + w) * 8) : make_uint4(0u, 0u, 0u, 0u);
          const unsigned x[4] = {raw[gr][w].x, raw[gr][w].y, raw[gr][w].z, raw[gr][w].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(x[i] << 16)), fabsf(__uint_as_float(x[i] & 0xFFFF0000u))));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int exponent = min(max((int)(__float_as_uint(most) >> 23), 6), 220);     // (biased) the power of two below the largest
      const float down = __uint_as_float((unsigned)(257 - exponent) << 23);           // brings it to [8, 16)
      const float up = __uint_as_float((unsigned)(exponent - 3 + (MASS ? 10 : 24)) << 23);   // and the scores back, the codes' powers of two included
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          const unsigned x[4] = {raw[gr][w].x, raw[gr][w].y, raw[gr][w].z, raw[gr][w].w};   // channels 0 1 | 2 3 | 4 5 | 6 7; wanted: 0 4 | 1 5 | 2 6 | 3 7
          float even[4], odd[4];   // channels 0 2 4 6 and 1 3 5 7
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            even[i] = __uint_as_float(x[i] << 16) * down;
            odd[i] = __uint_as_float(x[i] & 0xFFFF0000u) * down;
            sum += even[i] + odd[i];
            if (!MASS) odd[i] *= 0.0625f;
          }
          const __half2 pairs[4] = {__floats2half2_rn(even[0], even[2]), __floats2half2_rn(odd[0], odd[2]), __floats2half2_rn(even[1], even[3]), __floats2half2_rn(odd[1], odd[3])};
#pragma unroll
          for (int i = 0; i < 4; ++i) qb[nt][gr * STEPS + 2 * w + (i >> 1)][i & 1] = as_bits(pairs[i]);
        }
        if constexpr (!MASS) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
          for (int i = 0; i < 2; ++i) qsum[nt][gr][i] = -0x1p-24f * __shfl_sync(0xffffffffu, sum, 8 * t + 4 * i);   // of column 2 t + i: lanes 4 (2 t + i)
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        scale[nt][i] = p.scale_log2 * __shfl_sync(0xffffffffu, up, 8 * t + 4 * i);
        const int column = nt * 8 + 2 * t + i;
        limit[nt][i] = column < packed ? plan.length - plan.tokens + column / p.group : -1;
      }
    }
    const int sees_all = plan.length - plan.tokens;   // slots up to this one are seen by every token (of a row without a window)

    float o[MASS ? 1 : GROUPS][MASS ? 1 : MT][NT][4], top[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[nt][i] = NOTHING;
        sum[nt][i] = 0.f;
      }
    if constexpr (!MASS) {
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[gr][mt][nt][i] = 0.f;
    }
    // Of every group: the word from which on a step is larger than all so far; and, a byte each, the exponent of the power of two that brings its steps to the least group's.
    unsigned larger_from[GROUPS], down = 0x7F7F7F7Fu;
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) larger_from[gr] = 128u;

    for (int turn = 0; turn < tiles; ++turn) {
      copy_wait<STAGES - 1>();
      __syncwarp();
      const unsigned char* data = ring + (size_t)(warp * STAGES + stage_index) * S::STAGE_BYTES;
      stage_index ^= 1;
      const int key0 = (plan.first_tile + at + turn) * TILE + warp * WARP_KEYS;

      // Steps and zeros of the warp's keys, once for all lanes: a lane to a key.  A key whose values are not numbers gets a score that is not one: a weight of
      // zero times such a value would reach who does not see the key, a score that is chosen away does not.
      {
        const unsigned short* words = reinterpret_cast<const unsigned short*>(data + S::WORDS_AT) + lane * GROUPS;
        unsigned largest = 0u;
        if constexpr (!MASS) {
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) largest = max(largest, (unsigned)words[S::WORD_BYTES / 2 + gr]);
        }
        const bool bad = largest >= 0x7F80u;
        if constexpr (!MASS && GROUPS > 1) {
          bool larger = false;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) larger = larger || words[S::WORD_BYTES / 2 + gr] >= larger_from[gr];
          if (__any_sync(0xffffffffu, larger && !bad)) {   // rarely after the first tiles
            int step[GROUPS], least = 255, most = 0;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
              step[gr] = (int)max((larger_from[gr] >> 7) - 1u, __reduce_max_sync(0xffffffffu, bad ? 0u : (unsigned)words[S::WORD_BYTES / 2 + gr] >> 7));
              larger_from[gr] = (unsigned)(step[gr] + 1) << 7;
              if (step[gr]) least = min(least, step[gr]);
              most = max(most, step[gr]);
            }
            unsigned next = 0u;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
              const int old = (int)((down >> (8 * gr)) & 255u), now = 127 - max(0, min(MOST_APART, (step[gr] ? step[gr] : most) - least));   // (one of zeros: as the largest)
              next |= (unsigned)now << (8 * gr);
              if (now == old) continue;
              const float factor = __uint_as_float((unsigned)(127 + now - old) << 23);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[gr][mt][nt][i] *= factor;
            }
            down = next;
          }
        }
        int size = 0;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          const unsigned word = words[gr];
          const float step = bad ? __uint_as_float(0x7FC00000u) : word_step(word), zero = word_zero(word);
          key_scales[lane * GROUPS + gr] = make_float2(step, MASS ? __uint_as_float(as_bits(__float2half2_rn(zero * -0x1p-10f))) : step * zero);
          if constexpr (!MASS) {
            const unsigned value_word = words[S::WORD_BYTES / 2 + gr];
            const unsigned exponent = GROUPS > 1 ? (down >> (8 * gr)) & 255u : 127u;
            value_steps[lane * GROUPS + gr] = bad ? 0.f : word_step(value_word) * __uint_as_float(exponent << 23);
            size = max(size, (int)((value_word >> 7) + exponent));
            value_zeros[gr * WARP_KEYS + lane] = __float2half_rn(word_zero(value_word) * -0x1p-10f);
          }
        }
        if constexpr (!MASS) value_sizes[lane] = bad ? SMALLEST : fmaxf(SMALLEST, (float)(size - 254));
      }
      __syncwarp();

      // Scores of keys key0 + 16 h + g and + 8 (rows) for columns 2 t and 2 t + 1.
      float s[HALVES][NT][4];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][nt][i] = 0.f;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          unsigned low[WORDS], high[WORDS];   // of key g, of key g + 8
          const unsigned char* a = data + key_at[gr][0] + h * HALF_BYTES;
          const unsigned char* b = data + key_at[gr][1] + h * HALF_BYTES;
          if constexpr (WORDS == 1) {
            low[0] = *reinterpret_cast<const unsigned*>(a);
            high[0] = *reinterpret_cast<const unsigned*>(b);
          } else if constexpr (WORDS == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(a), y = *reinterpret_cast<const uint2*>(b);
            low[0] = x.x; low[1] = x.y; high[0] = y.x; high[1] = y.y;
          } else {
            const uint4 x = *reinterpret_cast<const uint4*>(a), y = *reinterpret_cast<const uint4*>(b);
            low[0] = x.x; low[1] = x.y; low[2] = x.z; low[3] = x.w;
            high[0] = y.x; high[1] = y.y; high[2] = y.z; high[3] = y.w;
          }
          float2 scaled[2];   // of key g, of key g + 8
          scaled[0] = key_scales[(16 * h + g) * GROUPS + gr];
          scaled[1] = key_scales[(16 * h + g + 8) * GROUPS + gr];
          float c[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[nt][i] = 0.f;
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            const unsigned low8 = low[w] >> 8, high8 = high[w] >> 8;
            unsigned a0, a1, a2, a3, b0, b1, b2, b3;
            if constexpr (MASS) {
              const __half2 low_away = as_half2(__float_as_uint(scaled[0].y)), high_away = as_half2(__float_as_uint(scaled[1].y));
              a0 = spread_values<0>(low[w], low8, low_away); a1 = spread_values<0>(high[w], high8, high_away);
              a2 = spread_values<1>(low[w], low8, low_away); a3 = spread_values<1>(high[w], high8, high_away);
              b0 = spread_values<2>(low[w], low8, low_away); b1 = spread_values<2>(high[w], high8, high_away);
              b2 = spread_values<3>(low[w], low8, low_away); b3 = spread_values<3>(high[w], high8, high_away);
            } else {
              a0 = spread<0>(low[w], low8); a1 = spread<0>(high[w], high8); a2 = spread<1>(low[w], low8); a3 = spread<1>(high[w], high8);
              b0 = spread<2>(low[w], low8); b1 = spread<2>(high[w], high8); b2 = spread<3>(low[w], low8); b3 = spread<3>(high[w], high8);
            }
            const int step = gr * STEPS + 2 * w;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_half(c[nt], a0, a1, a2, a3, qb[nt][step][0], qb[nt][step][1]);
              mma_half(c[nt], b0, b1, b2, b3, qb[nt][step + 1][0], qb[nt][step + 1][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (!MASS) s[h][nt][i] = fmaf(scaled[i >> 1].y, qsum[nt][gr][i & 1], s[h][nt][i]);
              s[h][nt][i] = fmaf(scaled[i >> 1].x, c[nt][i], s[h][nt][i]);
            }
        }
      }

      const bool masked = p.window > 0 || key0 + WARP_KEYS - 1 > sees_all;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][nt][i] *= scale[nt][i & 1];
      if (masked) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + 16 * h + g + 8 * (i >> 1), last = limit[nt][i & 1];
              const bool sees = key <= last && (p.window <= 0 || key > last - p.window);
              s[h][nt][i] = sees ? s[h][nt][i] : -INFINITY;
            }
      }
      if constexpr (MASS) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + 16 * h + g + 8 * (i >> 1), column = nt * 8 + 2 * t + (i & 1);
              if (column < packed && key < plan.length) p.scores[(((size_t)row * p.nkv + head) * p.score_columns + column) * p.most_slots + key] = s[h][nt][i];
            }
      }

      constexpr float lift = MASS ? 0.f : LIFT;
      float most[NT][2];   // of score + log2 of the values' size, less the lift
      bool grows = false;
      float size[HALVES][2];
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int half = 0; half < 2; ++half) size[h][half] = MASS ? 0.f : value_sizes[16 * h + g + 8 * half];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = fmaxf(s[0][nt][i] + size[0][0], s[0][nt][2 + i] + size[0][1]);
#pragma unroll
          for (int h = 1; h < HALVES; ++h) m = fmaxf(m, fmaxf(s[h][nt][i] + size[h][0], s[h][nt][2 + i] + size[h][1]));
          most[nt][i] = m - lift;
          grows = grows || most[nt][i] > top[nt][i] + RESCALE_STEP;
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float higher = fmaxf(top[nt][i], most[nt][i]);
            higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, 4));
            higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, 8));
            higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, 16));
            const float factor = ex2(top[nt][i] - higher);
            top[nt][i] = higher;
            sum[nt][i] *= factor;
            if constexpr (!MASS) {
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  o[gr][mt][nt][i] *= factor;
                  o[gr][mt][nt][2 + i] *= factor;
                }
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              s[h][nt][2 * half + i] = ex2(s[h][nt][2 * half + i] - top[nt][i]);
              sum[nt][i] += s[h][nt][2 * half + i];
            }
        }

      // Weighted values: channels (rows) by columns.
      if constexpr (!MASS) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) {
            unsigned pb[NT][2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float step = value_steps[(16 * h + g + 8 * half) * GROUPS + gr];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                pb[nt][half] = transpose8(as_bits(__floats2half2_rn(s[h][nt][2 * half] * step, s[h][nt][2 * half + 1] * step)));
              }
            }
            // The thread's channels of four keys: 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
            constexpr int LOADS = G == 128 ? 2 : 1;
            unsigned x[4][LOADS];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned char* from = data + value_at[gr][k] + h * HALF_BYTES;
              if constexpr (LOADS == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(from);
                x[k][0] = v.x;
                x[k][1] = v.y;
              } else {
                x[k][0] = *reinterpret_cast<const unsigned*>(from);
              }
            }
            const __half2 ab_away = *reinterpret_cast<const __half2*>(value_zeros + gr * WARP_KEYS + 16 * h + 2 * t);
            const __half2 cd_away = *reinterpret_cast<const __half2*>(value_zeros + gr * WARP_KEYS + 16 * h + 2 * t + 8);
#pragma unroll
            for (int m = 0; m < MT / 2; ++m) {   // four channels: half a word of each key
              const unsigned selector = G == 32 ? (g & 1 ? 0x7632 : 0x5410) : (m & 1 ? 0x7632 : 0x5410);
              const unsigned ab = __byte_perm(x[0][m >> 1], x[1][m >> 1], selector), cd = __byte_perm(x[2][m >> 1], x[3][m >> 1], selector);
              const unsigned ab8 = ab >> 8, cd8 = cd >> 8;
              const unsigned a0 = spread_values<0>(ab, ab8, ab_away), a1 = spread_values<1>(ab, ab8, ab_away), a2 = spread_values<0>(cd, cd8, cd_away), a3 = spread_values<1>(cd, cd8, cd_away);
              const unsigned b0 = spread_values<2>(ab, ab8, ab_away), b1 = spread_values<3>(ab, ab8, ab_away), b2 = spread_values<2>(cd, cd8, cd_away), b3 = spread_values<3>(cd, cd8, cd_away);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_half(o[gr][2 * m][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                mma_half(o[gr][2 * m + 1][nt], b0, b1, b2, b3, pb[nt][0], pb[nt][1]);
              }
            }
          }
      }
      __syncwarp();   // every lane has read the stage that is asked for next
      request();
    }

    // The warps' parts meet.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int column = nt * 8 + 2 * t + i;
        float all = sum[nt][i];
        all += __shfl_xor_sync(0xffffffffu, all, 4);
        all += __shfl_xor_sync(0xffffffffu, all, 8);
        all += __shfl_xor_sync(0xffffffffu, all, 16);
        if (g == 0) merge_sums[warp * COLUMNS + column] = make_float2(top[nt][i], all);
        if constexpr (!MASS) {
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) {
            float* to = merge_values + (size_t)(warp * COLUMNS + column) * D + gr * G + g * MINE;
            const float back = __uint_as_float((264u - (GROUPS > 1 ? (down >> (8 * gr)) & 255u : 127u)) << 23);   // 2^10, and the group's own size
#pragma unroll
            for (int mt = 0; mt < MT; mt += 2)
              *reinterpret_cast<float4*>(to + 2 * mt) = make_float4(back * o[gr][mt][nt][i], back * o[gr][mt][nt][2 + i], back * o[gr][mt + 1][nt][i], back * o[gr][mt + 1][nt][2 + i]);
          }
        }
      }
    __syncthreads();
    const bool whole = starts_here && ends_here;
    const size_t part = (size_t)blockIdx.x * 2 + (starts_here ? 1 : 0);
    for (int e = threadIdx.x; e < (MASS ? packed : packed * D); e += WARPS * 32) {
      const int column = MASS ? e : e / D, channel = MASS ? 0 : e % D;
      float2 sums[WARPS];
      float higher = NOTHING;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        sums[w] = merge_sums[w * COLUMNS + column];
        higher = fmaxf(higher, sums[w].x);
      }
      float value = 0.f, denominator = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float factor = ex2(sums[w].x - higher);   // (a sum that is not a number stays one)
        if (!MASS) value += merge_values[(size_t)(w * COLUMNS + column) * D + channel] * factor;
        denominator += sums[w].y * factor;
      }
      if (MASS) {
        if (whole) p.tops[((size_t)row * p.nkv + head) * p.score_columns + column] = make_float2(higher, 1.f / denominator);
        else p.part_sums[part * COLUMNS + column] = make_float2(higher, denominator);
      } else if (whole) {
        p.out[((size_t)(plan.first_token + column / p.group) * p.nq + head * p.group + column % p.group) * D + channel] = __float2bfloat16_rn(denominator == 0.f ? 0.f : value / denominator);
      } else {
        p.part_values[(part * COLUMNS + column) * D + channel] = value;
        if (channel == 0) p.part_sums[part * COLUMNS + column] = make_float2(higher, denominator);
      }
    }
    __syncthreads();   // the parts have been read
    tile += tiles;
  }
  copy_wait<0>();
}

// Joins the parts of a (row, KV head) that lies in several blocks' runs: a block to one of its columns.  D / 4 lanes share a column, four channels each; the
// others take parts side by side.
constexpr int JOIN_THREADS = 256, JOIN_LANES = D / 4, JOIN_SIDES = JOIN_THREADS / JOIN_LANES;
__global__ void __launch_bounds__(JOIN_THREADS) attention_packed_join_kernel(const PackedParams p, int columns) {
  extern __shared__ int starts[];
  __shared__ float4 values[JOIN_THREADS];
  __shared__ float warp_tops[JOIN_THREADS / 32];
  grid_dependency_wait();
  allow_dependents();
  make_plan(p, starts);
  const int row = blockIdx.z, head = blockIdx.y, lane = threadIdx.x % JOIN_LANES, side = threadIdx.x / JOIN_LANES;
  const int total = starts[p.rows], run = max(1, (total + p.blocks - 1) / p.blocks);
  const RowPlan plan = row_plan(p, row);
  if (plan.tiles == 0) return;
  const int first = starts[row] + head * plan.tiles, last = first + plan.tiles - 1;
  const int first_block = first / run, last_block = last / run;
  if (first_block == last_block) return;   // written by its block
  // Part number of block b: the stretch that begins the pair is its block's second, all others begin their block's run.
  auto part_of = [&](int b) { return ((size_t)b * 2 + (b == first_block ? 1 : 0)) * columns; };
  for (int column = blockIdx.x; column < plan.tokens * p.group; column += gridDim.x) {
    float higher = NOTHING;
    for (int b = first_block + threadIdx.x; b <= last_block; b += JOIN_THREADS) higher = fmaxf(higher, p.part_sums[part_of(b) + column].x);
    higher = warp_max(higher);
    if ((threadIdx.x & 31) == 0) warp_tops[threadIdx.x >> 5] = higher;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_THREADS / 32; ++w) higher = fmaxf(higher, warp_tops[w]);
    float4 value = make_float4(0.f, 0.f, 0.f, 0.f);
    float denominator = 0.f;
#pragma unroll 4
    for (int b = first_block + side; b <= last_block; b += JOIN_SIDES) {
      const size_t part = part_of(b) + column;
      const float2 s = p.part_sums[part];
      const float4 v = *reinterpret_cast<const float4*>(p.part_values + part * D + 4 * lane);
      const float factor = ex2(s.x - higher);
      value.x += v.x * factor; value.y += v.y * factor; value.z += v.z * factor; value.w += v.w * factor;
      denominator += s.y * factor;
    }
    values[threadIdx.x] = value;
    __shared__ float denominators[JOIN_SIDES];
    if (lane == 0) denominators[side] = denominator;
    __syncthreads();
    if (side == 0) {
#pragma unroll
      for (int i = 1; i < JOIN_SIDES; ++i) {
        const float4 v = values[i * JOIN_LANES + lane];
        value.x += v.x; value.y += v.y; value.z += v.z; value.w += v.w;
        denominator += denominators[i];
      }
      const float inverse = denominator == 0.f ? 0.f : 1.f / denominator;
      __nv_bfloat162 pairs[2] = {__floats2bfloat162_rn(value.x * inverse, value.y * inverse), __floats2bfloat162_rn(value.z * inverse, value.w * inverse)};
      *reinterpret_cast<uint2*>(p.out + ((size_t)(plan.first_token + column / p.group) * p.nq + head * p.group + column % p.group) * D + 4 * lane) = *reinterpret_cast<uint2*>(pairs);
    }
    __syncthreads();   // values and tops are free again
  }
}

// The same where there are more pairs than SMs, so that a pair has few parts: a warp to a column, all its channels, the parts one after another; no barriers.  (24 ragged rows
// of 40 / 8 heads, attention and join: 34.1 us; the other join with a block to a pair 38.  One row of 600 slots: 8.8 us with this one, 7.5 with a block to a column.)
__global__ void __launch_bounds__(JOIN_THREADS) attention_packed_join_few_kernel(const PackedParams p, int columns) {
  extern __shared__ int starts[];
  constexpr int VEC = D / 32;
  grid_dependency_wait();
  allow_dependents();
  make_plan(p, starts);
  const int row = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 31, column = blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
  const int total = starts[p.rows], run = max(1, (total + p.blocks - 1) / p.blocks);
  const RowPlan plan = row_plan(p, row);
  if (plan.tiles == 0 || column >= plan.tokens * p.group) return;
  const int first = starts[row] + head * plan.tiles, last = first + plan.tiles - 1;
  const int first_block = first / run, last_block = last / run;
  if (first_block == last_block) return;   // written by its block
  auto part_of = [&](int b) { return ((size_t)b * 2 + (b == first_block ? 1 : 0)) * columns + column; };
  float2 own = first_block + lane <= last_block ? p.part_sums[part_of(first_block + lane)] : make_float2(NOTHING, 0.f);   // most often all there are
  float higher = own.x;
  for (int b = first_block + 32 + lane; b <= last_block; b += 32) higher = fmaxf(higher, p.part_sums[part_of(b)].x);
  higher = warp_max(higher);
  float value[VEC] = {}, denominator = 0.f;
  for (int base = first_block; base <= last_block; base += 32) {
    if (base > first_block) own = base + lane <= last_block ? p.part_sums[part_of(base + lane)] : make_float2(NOTHING, 0.f);
    const float factor = ex2(own.x - higher);
    denominator += own.y * factor;
    const int count = min(32, last_block - base + 1);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const float weight = __shfl_sync(0xffffffffu, factor, i);
      const float* from = p.part_values + part_of(base + i) * D + VEC * lane;
      float v[VEC];
      if constexpr (VEC == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
#pragma unroll
      for (int c = 0; c < VEC; ++c) value[c] += v[c] * weight;
    }
  }
  denominator = warp_sum(denominator);
  const float inverse = denominator == 0.f ? 0.f : 1.f / denominator;
  __nv_bfloat162 pairs[VEC / 2];
#pragma unroll
  for (int c = 0; c < VEC / 2; ++c) pairs[c] = __floats2bfloat162_rn(value[2 * c] * inverse, value[2 * c + 1] * inverse);
  __nv_bfloat16* to = p.out + ((size_t)(plan.first_token + column / p.group) * p.nq + head * p.group + column % p.group) * D + VEC * lane;
  if constexpr (VEC == 4) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(pairs);
  else *reinterpret_cast<unsigned*>(to) = *reinterpret_cast<unsigned*>(pairs);
}

// Summed weights, second kernel: the kept scores become weights; four keys to a thread.
constexpr int ADD_THREADS = 128, ADD_KEYS = 4 * ADD_THREADS;
__global__ void __launch_bounds__(ADD_THREADS) packed_mass_add_kernel(const PackedParams p, int columns) {
  extern __shared__ int starts[];
  __shared__ float2 tops[16];
  grid_dependency_wait();
  allow_dependents();
  make_plan(p, starts);
  const int row = blockIdx.z, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const RowPlan plan = row_plan(p, row);
  if (plan.tiles == 0) return;
  const int packed = plan.tokens * p.group, old = p.kv_len[row] - (p.q_start[row + 1] - p.q_start[row]);
  const int total = starts[p.rows], run = max(1, (total + p.blocks - 1) / p.blocks);
  const int first = starts[row] + head * plan.tiles, last = first + plan.tiles - 1;
  const int first_block = first / run, last_block = last / run;
  const size_t pair = (size_t)row * p.nkv + head;
  const int* table = p.block_table + (size_t)row * p.table_width;
  // The slots of a thread's first keys and what they hold are asked for before the sums are there: one trip to memory behind another is what this kernel's time is.
  float* to[4];
  float before[4];
  auto ask = [&](int base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = base + i * ADD_THREADS + threadIdx.x;
      to[i] = nullptr;
      before[i] = 0.f;
      if (key >= plan.length) continue;
      const int logical = key / p.page_size, page = table[logical];
      if (page < 0 || page >= p.num_pages) continue;   // reported by the first kernel
      to[i] = p.mass + ((size_t)page * p.nkv + head) * p.page_size + (key - logical * p.page_size);
      if (key < old) before[i] = *to[i];
    }
  };
  ask(blockIdx.x * ADD_KEYS);
  if (first_block == last_block) {
    if ((int)threadIdx.x < packed) tops[threadIdx.x] = p.tops[pair * p.score_columns + threadIdx.x];
  } else {
    for (int column = warp; column < packed; column += ADD_THREADS / 32) {
      float higher = NOTHING, denominator = 0.f;
      for (int b = first_block + lane; b <= last_block; b += 32) higher = fmaxf(higher, p.part_sums[((size_t)b * 2 + (b == first_block ? 1 : 0)) * columns + column].x);
      higher = warp_max(higher);
      for (int b = first_block + lane; b <= last_block; b += 32) {
        const float2 s = p.part_sums[((size_t)b * 2 + (b == first_block ? 1 : 0)) * columns + column];
        denominator += s.y * ex2(s.x - higher);
      }
      denominator = warp_sum(denominator);
      if (lane == 0) tops[column] = make_float2(higher, 1.f / denominator);
    }
  }
  __syncthreads();
  for (int base = blockIdx.x * ADD_KEYS; base < plan.length; base += gridDim.x * ADD_KEYS) {
    if (base != (int)blockIdx.x * ADD_KEYS) ask(base);
    float added[4] = {0.f, 0.f, 0.f, 0.f};
    const float* from = p.scores + pair * p.score_columns * p.most_slots + base + threadIdx.x;
    for (int column = 0; column < packed; ++column) {
      const float2 top = tops[column];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = base + i * ADD_THREADS + threadIdx.x;
        const float score = key < plan.length ? from[(size_t)column * p.most_slots + i * ADD_THREADS] : -INFINITY;
        const float weight = ex2(score - top.x) * top.y;
        added[i] += score == -INFINITY ? 0.f : weight;   // (chosen away, not multiplied: the sum of a column may be no number)
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (to[i]) *to[i] = before[i] + added[i];
    }
  }
}

template <int G, int NT, bool MASS>
constexpr size_t packed_smem(int rows) {
  return (size_t)WARPS * (STAGES * Sizes<G, MASS>::STAGE_BYTES + Sizes<G, MASS>::SCALE_BYTES) + (size_t)WARPS * NT * 8 * ((MASS ? 0 : D * 4) + 8) + (size_t)(rows + 1) * 4;
}

template <int G, int NT, bool ALIGNED, bool MASS>
static int launch_packed(const PackedParams& p, cudaStream_t stream) {
  constexpr int MOST_ROWS = 1024;
  static bool ready[MAX_DEVICES] = {};
  bool& set = ready[current_device_slot()];
  if (!set) {
    const cudaError_t err = cudaFuncSetAttribute(attention_packed_kernel<G, NT, ALIGNED, MASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)packed_smem<G, NT, MASS>(MOST_ROWS));
    if (err != cudaSuccess) PYLON_REFUSE("paged_attention_packed: %s", cudaGetErrorString(err));
    set = true;
  }
  launch_dependent(attention_packed_kernel<G, NT, ALIGNED, MASS>, dim3(p.blocks), dim3(WARPS * 32), packed_smem<G, NT, MASS>(p.rows), stream, p);
  if (MASS) {
    const long long pairs = (long long)p.rows * p.nkv, wanted = (p.most_slots + ADD_KEYS - 1) / ADD_KEYS, fill = 1 + 16ll * multiprocessors() / pairs;
    launch_dependent(packed_mass_add_kernel, dim3((unsigned)(wanted < fill ? wanted : fill), p.nkv, p.rows), dim3(ADD_THREADS), (size_t)(p.rows + 1) * 4, stream, p, NT * 8);
    PYLON_CHECK_LAUNCH("attention_mass");
  }
  if ((long long)p.rows * p.nkv >= multiprocessors())
    launch_dependent(attention_packed_join_few_kernel, dim3(NT * 8 / (JOIN_THREADS / 32), p.nkv, p.rows), dim3(JOIN_THREADS), (size_t)(p.rows + 1) * 4, stream, p, NT * 8);
  else
    launch_dependent(attention_packed_join_kernel, dim3((unsigned)(p.group < NT * 8 ? p.group : NT * 8), p.nkv, p.rows), dim3(JOIN_THREADS), (size_t)(p.rows + 1) * 4, stream, p, NT * 8);
  PYLON_CHECK_LAUNCH("paged_attention_packed");
}

template <bool MASS>
static int launch_packed_for(const PackedParams& p, int channels, int columns, cudaStream_t stream) {
  const bool aligned = p.page_size % 16 == 0;
#define PYLON_PACKED(G)                                                                                                                     \
  if (channels == G) {                                                                                                                      \
    if (columns == 8) return aligned ? launch_packed<G, 1, true, MASS>(p, stream) : launch_packed<G, 1, false, MASS>(p, stream);             \
    return aligned ? launch_packed<G, 2, true, MASS>(p, stream) : launch_packed<G, 2, false, MASS>(p, stream);                               \
  }
  PYLON_PACKED(32)
  PYLON_PACKED(64)
#if PYLON_HEAD_DIM >= 128
  PYLON_PACKED(128)
#endif
  PYLON_REFUSE("paged_attention_packed: groups of %d channels of %d", channels, D);
}

static int check_packed(const char* name, const void* q, long long q_stride, const void* k_codes, const void* k_words, const void* v_codes, const void* v_words, int table_width, int page_size,
                        int num_pages, int nq, int nkv, int window, int rows, int blocks, int packed, const int* error, const float* scratch) {
  if (nkv < 1 || nq < 1 || nq % nkv || nkv > 65535 || page_size < 1 || table_width < 1 || num_pages < 1 || window < 0 || rows > 1024 || blocks < 1 || packed < 1 || packed > SMALL_ROWS)
    PYLON_REFUSE("%s: heads %d/%d, page size %d, table width %d, window %d, %d rows, %d blocks, %d packed", name, nq, nkv, page_size, table_width, window, rows, blocks, packed);
  if ((long long)table_width * page_size > 0x7FFFFFFF - 4096) PYLON_REFUSE("%s: %d pages of %d slots to a row", name, table_width, page_size);
  if ((uintptr_t)q % 16 || q_stride % 8 || (uintptr_t)k_codes % 16 || (uintptr_t)v_codes % 16 || (uintptr_t)k_words % 16 || (uintptr_t)v_words % 16)
    PYLON_REFUSE("%s: q and pages must be 16-byte aligned, the rows of q a multiple of 8 elements apart", name);
  if (!error || !scratch) PYLON_REFUSE("%s: an error word and scratch memory are needed", name);
  return 0;
}

}  // namespace pylon

using namespace pylon;

// Blocks of a launch for rows of at most `packed` packed query rows, and the floats of scratch memory they need.
// How many blocks the device has room for at once: what a launch's runs are cut for.
template <int G, int NT, bool MASS>
static int resident_blocks(int rows) {
  const int fit = (int)(228 * 1024 / (packed_smem<G, NT, MASS>(rows) + 1024)), most = blocks_an_sm(NT, MASS);   // 1 KB of a block's shared memory is the system's
  return multiprocessors() * (fit < most ? fit : most);
}
extern "C" int pylon_attention_packed_blocks(int packed, int group, int rows, int mass) {
  if (rows > 1024) return 0;
#define PYLON_PACKED_BLOCKS(G)                                                                                   \
  if (group == G) {                                                                                              \
    if (packed <= 8) return mass ? resident_blocks<G, 1, true>(rows) : resident_blocks<G, 1, false>(rows);       \
    return mass ? resident_blocks<G, 2, true>(rows) : resident_blocks<G, 2, false>(rows);                        \
  }
  PYLON_PACKED_BLOCKS(32)
  PYLON_PACKED_BLOCKS(64)
#if PYLON_HEAD_DIM >= 128
  PYLON_PACKED_BLOCKS(128)
#endif
  return 0;
}
extern "C" long long pylon_attention_packed_scratch_floats(int blocks, int packed) { return (long long)blocks * 2 * (packed <= 8 ? 8 : 16) * (D + 2); }
extern "C" long long pylon_packed_mass_scratch_floats(int blocks, int packed, int rows, int nkv, int max_kv) {
  return (long long)blocks * 2 * (packed <= 8 ? 8 : 16) * 2 + (long long)rows * nkv * packed * (2ll + max_kv);
}

// packed: tokens x query heads of a KV head of the longest row that is not skipped (8 or fewer: a column tile of 8, else of 16).
extern "C" int pylon_attention_packed(const void* q, long long q_stride, const void* k_codes, const void* k_words, const void* v_codes, const void* v_words, void* out, float* scratch,
                                      const int* q_start, const int* kv_len, const int* block_table, int table_width, int page_size, int num_pages, int nq, int nkv, int group, int window,
                                      float scale, int rows, int blocks, int packed, int* error, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (int code = check_packed("paged_attention_packed", q, q_stride, k_codes, k_words, v_codes, v_words, table_width, page_size, num_pages, nq, nkv, window, rows, blocks, packed, error, scratch))
    return code;
  PackedParams p = {};
  p.q = (const __nv_bfloat16*)q; p.q_stride = q_stride;
  p.k_codes = (const unsigned char*)k_codes; p.k_words = (const unsigned short*)k_words;
  p.v_codes = (const unsigned char*)v_codes; p.v_words = (const unsigned short*)v_words;
  p.out = (__nv_bfloat16*)out; p.q_start = q_start; p.kv_len = kv_len; p.block_table = block_table;
  p.table_width = table_width; p.page_size = page_size; p.num_pages = num_pages; p.nq = nq; p.nkv = nkv; p.group = nq / nkv; p.window = window; p.rows = rows; p.blocks = blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int columns = packed <= 8 ? 8 : 16;
  p.part_values = scratch;
  p.part_sums = reinterpret_cast<float2*>(scratch + (size_t)blocks * 2 * columns * D);
  p.error = error;
  p.last = 0x7FFFFFFF;
  p.most_packed = packed;
  p.most_slots = table_width * page_size;
  return launch_packed_for<false>(p, group, columns, stream);
}

// Summed weights of rows whose last `last` tokens are at most `packed` packed query rows; no row's slots from max_kv on are looked at.
extern "C" int pylon_packed_mass(const void* q, long long q_stride, const void* k_codes, const void* k_words, float* mass, float* scratch, const int* q_start, const int* kv_len,
                                 const int* block_table, int table_width, int page_size, int num_pages, int nq, int nkv, int group, int rows, int last, int max_kv, float scale, int blocks,
                                 int packed, int* error, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (int code = check_packed("attention_mass", q, q_stride, k_codes, k_words, k_codes, k_words, table_width, page_size, num_pages, nq, nkv, 0, rows, blocks, packed, error, scratch)) return code;
  if (last < 1 || (long long)last * (nq / nkv) > packed || max_kv < 1) PYLON_REFUSE("attention_mass: %d votes of %d packed query rows, longest row %d", last, packed, max_kv);
  PackedParams p = {};
  p.q = (const __nv_bfloat16*)q; p.q_stride = q_stride;
  p.k_codes = (const unsigned char*)k_codes; p.k_words = (const unsigned short*)k_words;
  p.q_start = q_start; p.kv_len = kv_len; p.block_table = block_table;
  p.table_width = table_width; p.page_size = page_size; p.num_pages = num_pages; p.nq = nq; p.nkv = nkv; p.group = nq / nkv; p.rows = rows; p.blocks = blocks;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int columns = packed <= 8 ? 8 : 16;
  p.part_sums = reinterpret_cast<float2*>(scratch);
  p.tops = p.part_sums + (size_t)blocks * 2 * columns;
  p.scores = reinterpret_cast<float*>(p.tops + (size_t)rows * nkv * packed);
  p.score_columns = packed;
  p.error = error;
  p.mass = mass;
  p.last = last;
  p.most_packed = packed;
  p.most_slots = max_kv < table_width * page_size ? max_kv : table_width * page_size;
  return launch_packed_for<true>(p, group, columns, stream);
}
