// The sums of attention weights of attention_mass.cu for prompt portions, on the fifth-generation tensor cores: bfloat16 queries, keys in plain bfloat16 pages
// or in the 4-bit pages of packed_cache.cu (whose values are bfloat16 numbers exactly).
//
// Built for one head size per library: -DPYLON_HEAD_DIM=64 or 128.
//
// Two passes over the keys, since a weight needs its whole row's sum.  Both take a (row, KV head)'s packed queries (token x query head) 256 at a time, laid
// out in shared memory once, and stream 128-key tiles past them; they differ in who is a row of the product, which is a lane of tensor memory and so a thread:
//   first pass    S = Q K^T, queries are rows (two products of 128 x 128): a thread keeps maximum and sum of its query over a stretch of tiles - no shuffles;
//   second pass   S = K Q^T, keys are rows (128 x 256): a thread adds up exp2(score - maximum) / sum of its key over the queries - no shuffles either, and
//                 every mass has one owner that adds in a fixed order.
// 25 warps: 16 of softmax (four warpgroups, each 64 scores of a row; two warpgroups with 128 took 45 us where these take 41), 8 that bring keys (copies of 16
// bytes, or codes that become bfloat16 numbers on the way; four took 295 us over 131,072 packed keys where eight take 280) into a ring of three tiles in the 128-byte swizzle, one that
// issues the products into two score buffers (2 x 256 columns: all of tensor memory; one block to an SM).
// What its time goes by: both passes need one exponential per score (16 a clock and SM, twice what the products take), and run at half that rate (issue slots 54 and 45 %), by the latencies of
// its loads of tensor memory and of its first tile (a pass over 500 keys takes 9 us).  64 voting tokens of 32 / 8 heads of 128: 41 us over 16,384 plain keys and 44 over
// packed ones (96 and 94 for attention_mass_mma.cu's m16n8k16 products, whose rate bounds them), 262 and 280 over 131,072 (660 and 643).
//
// Work.  The tiles of all rows are cut into stretches of equal length, the least that gives no more stretches than the device has SMs (at most 16 tiles); the
// plan is made on the device from the rows' lengths, by both passes alike.  A stretch's maxima and sums lie in scratch memory under its number; the second pass
// joins those of a (row, KV head) itself, all blocks in the same order.
//
// Waits on mbarriers are bounded: one that runs out sets the error word (1 keys, 2 products, 3 softmax) and every role goes on to the end without waiting again.
#include "common.cuh"

#ifndef PYLON_HEAD_DIM
#define PYLON_HEAD_DIM 128
#endif

namespace pylon {

constexpr int D = PYLON_HEAD_DIM;
static_assert(D == 64 || D == 128, "built for head sizes 64 and 128");
constexpr int CHUNK = 256, TILE = 128, STAGES = 3, MOST_TILES = 16;
constexpr int SOFT_WARPS = 16, SOFT_THREADS = SOFT_WARPS * 32, LOAD_THREADS = 256, THREADS = SOFT_THREADS + LOAD_THREADS + 32;
constexpr int Q_PANEL = CHUNK * 128, K_PANEL = TILE * 128;      // 64 channels of all rows
constexpr int Q_BYTES = CHUNK * D * 2, K_BYTES = TILE * D * 2;
constexpr int UNITS = D / 8;                                    // 16-byte units of a row
constexpr unsigned WAIT_LIMIT = 1u << 22;
constexpr float NOTHING = -1.0e30f;                             // a maximum before any score (times any scale below 10^8 still a number)
constexpr float RESCALE_STEP = 8.f;                             // log2: the reference of a sum moves when a score is more than this above it
constexpr int MOST_ROWS = 1024;
constexpr int ISSUER = SOFT_WARPS + LOAD_THREADS / 32;          // the warp that issues the products

struct Shared {
  unsigned char q[Q_BYTES];
  unsigned char keys[STAGES][K_BYTES];
  long long offsets[2][TILE];          // where a tile's keys lie (rows of the pages), -1: nowhere
  float2 tops[CHUNK];                  // second pass: minus the scaled maximum (log2), 1 / sum; first pass: maximum and sum over the second half of every tile
  int limits[CHUNK];                   // second pass: the last slot that a column sees
  float added[4][MOST_TILES * TILE];   // second pass: the warpgroups' sums
  int starts[MOST_ROWS + 1];
  uint64_t k_full[STAGES], k_empty[STAGES], s_full[2], s_empty[2];
  unsigned tmem;
  int stretch_tiles, dead;
};
constexpr size_t SMEM = sizeof(Shared) > 120 * 1024 ? sizeof(Shared) : 120 * 1024;   // never two blocks on an SM: each takes all of tensor memory
static_assert(SMEM <= 227 * 1024, "shared memory");

struct MassParams {
  const __nv_bfloat16* q;
  long long q_stride;
  const void* keys;
  const unsigned short* words;    // 4-bit pages: their words, channels to a group; null for plain pages
  int group;
  float* mass;
  const int* q_start;
  const int* kv_len;
  const int* block_table;
  int table_width, page_size, num_pages, nq, nkv, heads /* of a KV head */, rows, last, most_slots, columns;
  float scale_log2;
  float2* parts;                  // [stretches of all rows][columns]: maximum of the unscaled scores, sum
  int* error;
};

__device__ __forceinline__ unsigned smem_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint64_t* bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_address(bar)), "r"(count)); }
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_address(bar)) : "memory"); }
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, unsigned parity) {
  for (unsigned tries = 0; tries < WAIT_LIMIT; ++tries) {
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_address(bar)), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ void issue_mma(unsigned tmem_d, uint64_t a_desc, uint64_t b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_load_32(unsigned taddr, float (&x)[32]) {
  unsigned r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
}
// K-major operands in the 128-byte swizzle: rows of 128 bytes, 1,024 bytes from eight rows to the next eight.
__device__ __forceinline__ uint64_t operand(unsigned address) {
  return (uint64_t)((address & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16: bfloat16 operands, float32 results.
constexpr unsigned instruction(int m, int n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct MassRow {
  int first, votes, new_tokens, length, columns, tiles;
};
__device__ __forceinline__ MassRow mass_row(const MassParams& p, int row) {
  MassRow r;
  r.new_tokens = p.q_start[row + 1] - p.q_start[row];
  r.length = min(p.kv_len[row], p.most_slots);
  r.votes = r.length > 0 ? min(r.new_tokens, p.last) : 0;
  r.first = p.q_start[row] + r.new_tokens - r.votes;
  r.columns = r.votes * p.heads;
  r.tiles = r.votes > 0 ? (r.length + TILE - 1) / TILE : 0;
  return r;
}

// By warp 0: the stretches' length, and starts[r], the stretches before row r; starts[rows] of them in all.
__device__ __forceinline__ void make_plan(const MassParams& p, Shared& s) {
  const int lane = threadIdx.x;
  int* row_tiles = reinterpret_cast<int*>(s.added);
  long long tiles = 0;
  for (int row = lane; row < p.rows; row += 32) {   // each lane reads back its own
    row_tiles[row] = mass_row(p, row).tiles;
    tiles += (long long)row_tiles[row] * p.nkv;
  }
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, offset);
  int stretch = (int)min((long long)MOST_TILES, max(1ll, (tiles + gridDim.x - 1) / gridDim.x));
  for (;; ++stretch) {
    int before = 0;
    for (int base = 0; base < p.rows; base += 32) {
      const int row = base + lane;
      const int own = row < p.rows ? (row_tiles[row] + stretch - 1) / stretch * p.nkv : 0;
      int upto = own;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += other;
      }
      if (row < p.rows) s.starts[row] = before + upto - own;
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (before <= (int)gridDim.x || stretch >= MOST_TILES) {
      if (lane == 0) {
        s.starts[p.rows] = before;
        s.stretch_tiles = stretch;
      }
      break;
    }
  }
}

__device__ __forceinline__ uint4 unpack8(unsigned codes, unsigned word) {   // eight channels as bfloat16: 16 + code behind the exponent of 16, then exact arithmetic
  const unsigned step_bits = (word & 0xFFF0u) * 0x00010001u;
  const __nv_bfloat162 away = __float2bfloat162_rn((float)(16 + (int)(word & 15u))), step = *reinterpret_cast<const __nv_bfloat162*>(&step_bits);
  unsigned pairs[4];   // channels 0 4 | 1 5 | 2 6 | 3 7
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned number = ((i ? codes >> (4 * i - 3) : codes << 3) & 0x00780078u) | 0x41804180u;
    const __nv_bfloat162 value = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&number), away), step);
    pairs[i] = *reinterpret_cast<const unsigned*>(&value);
  }
  return make_uint4(__byte_perm(pairs[0], pairs[1], 0x5410), __byte_perm(pairs[2], pairs[3], 0x5410), __byte_perm(pairs[0], pairs[1], 0x7632), __byte_perm(pairs[2], pairs[3], 0x7632));
}

// (maximum of the unscaled scores, sum) of two sets of keys.
__device__ __forceinline__ float2 join(float2 a, float2 b, float scale_log2) {
  const float top = fmaxf(a.x, b.x);
  return make_float2(top, a.y * ex2((a.x - top) * scale_log2) + b.y * ex2((b.x - top) * scale_log2));   // (a sum that is not a number stays one)
}

__device__ __forceinline__ void loaders_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(LOAD_THREADS) : "memory"); }

template <bool ADD, bool PACKED>
__global__ void __launch_bounds__(THREADS, 1) mass_tcgen05_kernel(const MassParams p) {
  extern __shared__ __align__(1024) unsigned char dynamic[];
  Shared& s = *reinterpret_cast<Shared*>(dynamic);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Tensor memory is asked for only when the kernel ahead has ended, and dependents start only when it is there: nobody who holds some waits for someone who needs it.
  grid_dependency_wait();
  if ((smem_address(dynamic) & 1023u) != 0) {   // the swizzle's arithmetic assumes it
    if (threadIdx.x == 0) atomicExch(p.error, 4);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { barrier_init(&s.k_full[i], LOAD_THREADS); barrier_init(&s.k_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { barrier_init(&s.s_full[i], 1); barrier_init(&s.s_empty[i], SOFT_THREADS); }
    s.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_address(&s.tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  if (warp == 0) make_plan(p, s);
  fence_before();
  __syncthreads();
  fence_after();
  allow_dependents();
  const unsigned tmem = s.tmem;
  const int stretch_tiles = s.stretch_tiles, total = s.starts[p.rows];
  const float slack = RESCALE_STEP / p.scale_log2;
  int turn = 0;   // tiles before this one, of all stretches and chunks: the barriers' phases follow it
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    int row = 0;
    for (int high = p.rows - 1; row < high;) {
      const int middle = (row + high + 1) >> 1;
      if (s.starts[middle] <= item) row = middle;
      else high = middle - 1;
    }
    const MassRow r = mass_row(p, row);
    const int stretches = (r.tiles + stretch_tiles - 1) / stretch_tiles, within = item - s.starts[row], head = within / stretches, place = within - head * stretches;
    const int first_tile = place * stretch_tiles, tiles = min(stretch_tiles, r.tiles - first_tile);
    const int all_see = r.length - r.votes;   // slots up to this one are seen by every voting token
    const int* table = p.block_table + (size_t)row * p.table_width;
    for (int column0 = 0; column0 < r.columns; column0 += CHUNK) {
      const int columns = min(CHUNK, r.columns - column0);
      float top = NOTHING, sum[4] = {0.f, 0.f, 0.f, 0.f};
      if (warp < SOFT_WARPS) {
        // Queries: rows of the operand, zeros behind the last one.  Every product of the chunk before has been waited for, and the warps that bring keys are at it
        // already.  All loads of a thread are in flight at once: one after another they were a third of the kernel's time.
        constexpr int AT_ONCE = CHUNK * UNITS / SOFT_THREADS;
        {
          uint4 v[AT_ONCE];
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i) {
            const int e = threadIdx.x + i * SOFT_THREADS, n = e / UNITS, c = e % UNITS, column = column0 + n, token = column / p.heads;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (n < columns) v[i] = *reinterpret_cast<const uint4*>(p.q + (size_t)(r.first + token) * p.q_stride + (size_t)(head * p.heads + column - token * p.heads) * D + c * 8);
          }
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i) {
            const int e = threadIdx.x + i * SOFT_THREADS, n = e / UNITS, c = e % UNITS;
            *reinterpret_cast<uint4*>(s.q + (c / 8) * Q_PANEL + n * 128 + (((c % 8) ^ (n & 7)) << 4)) = v[i];
          }
        }
        if (ADD && threadIdx.x < CHUNK) {
          const int n = threadIdx.x, column = column0 + n;
          float2 all = make_float2(NOTHING, 0.f);
          if (n < columns) {
            const float2* from = p.parts + (size_t)(s.starts[row] + head * stretches) * p.columns + column;
#pragma unroll 1
            for (int base = 0; base < stretches; base += 8) {
              float2 part[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) part[i] = base + i < stretches ? from[(size_t)(base + i) * p.columns] : make_float2(NOTHING, 0.f);
#pragma unroll
              for (int i = 0; i < 8; ++i) all = join(all, part[i], p.scale_log2);
            }
          }
          s.tops[n] = n < columns ? make_float2(-all.x * p.scale_log2, 1.f / all.y) : make_float2(0.f, 0.f);
          s.limits[n] = n < columns ? r.length - r.votes + column / p.heads : -1;
        }
        fence_async_shared();
      }
      if (warp < SOFT_WARPS || warp == ISSUER) asm volatile("bar.sync 2, %0;\n" ::"n"(SOFT_THREADS + 32) : "memory");   // softmax and products; who brings keys needs none of this
      bool alive = *reinterpret_cast<volatile int*>(&s.dead) == 0;   // (not the same for all threads: who is not alive takes every turn, but waits for nothing)

      if (warp >= SOFT_WARPS && warp < ISSUER) {
        // ---- keys ----
        const int tid = threadIdx.x - SOFT_THREADS;
        auto locate = [&](int tile, int buffer) {   // a thread to a key; the loaders meet before they are used
          if (tid >= TILE) return;
          const int key = (first_tile + tile) * TILE + tid;
          long long at = -1;
          if (tile < tiles && key < r.length) {
            const int logical = key / p.page_size, page = table[logical];
            if (page >= 0 && page < p.num_pages) at = ((long long)page * p.nkv + head) * p.page_size + (key - logical * p.page_size);
            else if (!ADD) atomicExch(p.error, PYLON_ERROR_BAD_PAGE);
          }
          s.offsets[buffer][tid] = at;
        };
        if constexpr (PACKED) {
          constexpr int KEYS_AT_ONCE = LOAD_THREADS / UNITS, PIECES = TILE / KEYS_AT_ONCE;   // a thread has the same unit of PIECES keys
          const int c = tid % UNITS, first_key = tid / UNITS, words_row = D / p.group, word_at = c * 8 / p.group;
          const unsigned* codes = reinterpret_cast<const unsigned*>(p.keys);
          unsigned next_codes[PIECES];
          unsigned short next_words[PIECES];
          auto fetch = [&](int buffer) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const long long at = s.offsets[buffer][first_key + i * KEYS_AT_ONCE];
              next_codes[i] = at >= 0 ? codes[at * UNITS + c] : 0u;
              next_words[i] = at >= 0 ? p.words[at * words_row + word_at] : (unsigned short)0;
            }
          };
          locate(0, 0);
          loaders_sync();
          fetch(0);
          for (int t = 0; t < tiles; ++t) {
            const int stage = (turn + t) % STAGES;
            locate(t + 1, (t + 1) & 1);
            if (alive && !barrier_wait(&s.k_empty[stage], (((turn + t) / STAGES) & 1) ^ 1)) { atomicExch(p.error, 1); s.dead = 1; alive = false; }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              const int key = first_key + i * KEYS_AT_ONCE;
              *reinterpret_cast<uint4*>(s.keys[stage] + (c / 8) * K_PANEL + key * 128 + (((c % 8) ^ (key & 7)) << 4)) = unpack8(next_codes[i], next_words[i]);
            }
            fence_async_shared();
            barrier_arrive(&s.k_full[stage]);
            loaders_sync();
            fetch((t + 1) & 1);
          }
        } else {
          const __nv_bfloat16* keys = reinterpret_cast<const __nv_bfloat16*>(p.keys);
          auto ask = [&](int t) {
            const int stage = (turn + t) % STAGES;
            if (alive && !barrier_wait(&s.k_empty[stage], (((turn + t) / STAGES) & 1) ^ 1)) { atomicExch(p.error, 1); s.dead = 1; alive = false; }
            locate(t, t & 1);
            loaders_sync();
            const unsigned base = smem_address(s.keys[stage]);
#pragma unroll
            for (int e = tid; e < TILE * UNITS; e += LOAD_THREADS) {
              const int key = e / UNITS, c = e % UNITS;
              const long long at = s.offsets[t & 1][key];
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                           ::"r"(base + (c / 8) * K_PANEL + key * 128 + (((c % 8) ^ (key & 7)) << 4)), "l"(keys + max(at, 0ll) * D + c * 8), "r"(at >= 0 ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
          };
          for (int t = 0; t <= tiles; ++t) {   // one tile on its way while the one before lands
            if (t < tiles) ask(t);
            if (t == 0) continue;
            if (t < tiles) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            else asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            fence_async_shared();
            barrier_arrive(&s.k_full[(turn + t - 1) % STAGES]);
          }
        }
      } else if (warp == ISSUER) {
        // ---- products ----
        if (lane == 0) {
          const unsigned q_base = smem_address(s.q);
          for (int t = 0; t < tiles && alive; ++t) {
            const int stage = (turn + t) % STAGES, buffer = (turn + t) & 1;
            if (!barrier_wait(&s.k_full[stage], ((turn + t) / STAGES) & 1) || !barrier_wait(&s.s_empty[buffer], (((turn + t) >> 1) & 1) ^ 1)) {
              atomicExch(p.error, 2);
              s.dead = 1;
              alive = false;
              break;
            }
            fence_after();
            const unsigned k_base = smem_address(s.keys[stage]);
            if constexpr (ADD) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)   // 16 channels: 32 bytes along the swizzled row; 64 to a panel
                issue_mma(tmem + buffer * 256, operand(k_base + (kk / 4) * K_PANEL) + 2 * (kk % 4), operand(q_base + (kk / 4) * Q_PANEL) + 2 * (kk % 4),
                          columns > 128 ? instruction(128, 256) : instruction(128, 128), kk != 0 ? 1u : 0u);
            } else {
              for (int half = 0; half * 128 < columns; ++half)
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                  issue_mma(tmem + buffer * 256 + half * 128, operand(q_base + (kk / 4) * Q_PANEL + half * 128 * 128) + 2 * (kk % 4), operand(k_base + (kk / 4) * K_PANEL) + 2 * (kk % 4),
                            instruction(128, 128), kk != 0 ? 1u : 0u);
            }
            commit(&s.k_empty[stage]);
            commit(&s.s_full[buffer]);
          }
        }
      } else {
        // ---- softmax ----
        const int half = (warp >> 2) & 1, side = warp >> 3, own = (warp & 3) * 32 + lane;   // 128 queries of 256; 64 scores of 128; lane of tensor memory
        const int first_score = half * 128 + side * 64;
        const bool mine = (ADD ? first_score : half * 128) < columns;
        const unsigned lane_base = tmem + ((unsigned)((warp & 3) * 32) << 16) + first_score;
        const int limit = r.length - r.votes + (column0 + half * 128 + own) / p.heads;   // first pass: the last slot that the thread's query sees
        alive = __all_sync(0xffffffffu, alive);
        for (int t = 0; t < tiles && alive; ++t) {
          const int buffer = (turn + t) & 1, key0 = (first_tile + t) * TILE;
          alive = __all_sync(0xffffffffu, barrier_wait(&s.s_full[buffer], ((turn + t) >> 1) & 1));   // loads of tensor memory are a whole warp's
          if (!alive) {
            atomicExch(p.error, 3);
            s.dead = 1;
            break;
          }
          fence_after();
          const bool some_hidden = key0 + TILE - 1 > all_see || (ADD && first_score + 64 > columns);
          if (ADD) sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll 1
          for (int part = 0; mine && part < 2; ++part) {
            float c[32];
            tmem_load_32(lane_base + buffer * 256 + part * 32, c);
            if constexpr (ADD) {
              const float4* tops = reinterpret_cast<const float4*>(s.tops + first_score + part * 32);
              if (some_hidden) {   // what a column does not see is chosen away, not multiplied: a column's sum may be no number
                const int* limits = s.limits + first_score + part * 32;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float2 at = s.tops[first_score + part * 32 + i];
                  const float weight = ex2(fmaf(c[i], p.scale_log2, at.x)) * at.y;
                  sum[i & 3] += key0 + own <= limits[i] ? weight : 0.f;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float4 two = tops[i];
                  sum[(2 * i) & 3] = fmaf(ex2(fmaf(c[2 * i], p.scale_log2, two.x)), two.y, sum[(2 * i) & 3]);
                  sum[(2 * i + 1) & 3] = fmaf(ex2(fmaf(c[2 * i + 1], p.scale_log2, two.z)), two.w, sum[(2 * i + 1) & 3]);
                }
              }
            } else {
              if (some_hidden) {
#pragma unroll
                for (int i = 0; i < 32; ++i) c[i] = key0 + side * 64 + part * 32 + i <= limit ? c[i] : -INFINITY;
              }
              float four[4] = {c[0], c[1], c[2], c[3]};   // (one chain of maxima would be as long as the exponentials take)
#pragma unroll
              for (int i = 4; i < 32; ++i) four[i & 3] = fmaxf(four[i & 3], c[i]);
              const float most = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3]));
              if (most > top + slack) {
                const float down = ex2((top - most) * p.scale_log2);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] *= down;
                top = most;
              }
              const float away = -p.scale_log2 * top;
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[i & 3] += ex2(fmaf(c[i], p.scale_log2, away));
            }
          }
          fence_before();
          barrier_arrive(&s.s_empty[buffer]);
          if (ADD) {
            float* to = &s.added[warp >> 2][t * TILE + own];
            const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            *to = column0 ? *to + all : all;
          }
        }
        if (!ADD && side) s.tops[half * 128 + own] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
      }
      turn += tiles;
      __syncthreads();   // queries and tops are free again
      if (!ADD && threadIdx.x < CHUNK && (int)threadIdx.x < columns)
        p.parts[(size_t)item * p.columns + column0 + threadIdx.x] = join(make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3])), s.tops[threadIdx.x], p.scale_log2);
    }
    if (ADD) {
      for (int i = threadIdx.x; i < tiles * TILE; i += THREADS) {
        const int key = first_tile * TILE + i;
        if (key >= r.length) break;
        const int logical = key / p.page_size, page = table[logical];
        if (page < 0 || page >= p.num_pages) continue;   // reported by the first pass
        float* to = p.mass + ((size_t)page * p.nkv + head) * p.page_size + (key - logical * p.page_size);
        *to = (key < r.length - r.new_tokens ? *to : 0.f) + ((s.added[0][i] + s.added[1][i]) + (s.added[2][i] + s.added[3][i]));
      }
      __syncthreads();
    }
  }
  fence_before();
  __syncthreads();
  if (warp == ISSUER) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
}

template <bool ADD, bool PACKED>
static int launch_pass(const MassParams& p, int blocks, cudaStream_t stream) {
  static bool ready[MAX_DEVICES] = {};
  bool& set = ready[current_device_slot()];
  if (!set) {
    const cudaError_t err = cudaFuncSetAttribute(mass_tcgen05_kernel<ADD, PACKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
    if (err != cudaSuccess) PYLON_REFUSE("attention_mass: %s", cudaGetErrorString(err));
    set = true;
  }
  launch_dependent(mass_tcgen05_kernel<ADD, PACKED>, dim3(blocks), dim3(THREADS), SMEM, stream, p);
  return 0;
}

// The most stretches of all rows: no more than SMs, or of the greatest length.
static long long most_stretches(int rows, int nkv, int max_kv) {
  const long long longest = (long long)rows * nkv * ((max_kv + MOST_TILES * TILE - 1) / (MOST_TILES * TILE));
  return longest > multiprocessors() ? longest : multiprocessors();
}

}  // namespace pylon

using namespace pylon;

extern "C" long long pylon_attention_mass_tcgen05_scratch_floats(int rows, int nkv, int max_kv, int columns) { return 2 * most_stretches(rows, nkv, max_kv) * columns; }

// keys: plain bfloat16 pages (words null) or codes.  columns: the most packed queries of a row, min(last, longest row) * nq / nkv.  max_kv: no row's
// slots from max_kv on are looked at.
extern "C" int pylon_attention_mass_tcgen05(const void* q, long long q_stride, const void* keys, const void* words, float* mass, float* scratch, const int* q_start, const int* kv_len,
                                            const int* block_table, int table_width, int page_size, int num_pages, int nq, int nkv, int group, int rows, int last, int max_kv, float scale,
                                            int* error, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (nkv < 1 || nkv > 65535 || nq < 1 || nq % nkv || page_size < 1 || table_width < 1 || num_pages < 1 || last < 1 || max_kv < 1 || rows > MOST_ROWS)
    PYLON_REFUSE("attention_mass: heads %d/%d, page size %d, %d rows, %d votes", nq, nkv, page_size, rows, last);
  if ((long long)table_width * page_size > 0x7FFFFFFF - 4096) PYLON_REFUSE("attention_mass: %d pages of %d slots to a row", table_width, page_size);
  if ((uintptr_t)q % 16 || q_stride % 8 || (uintptr_t)keys % 16) PYLON_REFUSE("attention_mass: q and pages must be 16-byte aligned, the rows of q a multiple of 8 elements apart");
  if (words && ((group != 32 && group != 64 && group != 128) || D % group)) PYLON_REFUSE("attention_mass: groups of %d channels of %d", group, D);
  if (!error || !scratch) PYLON_REFUSE("attention_mass: an error word and scratch memory are needed");
  const long long columns = (long long)last * (nq / nkv);
  if (columns > 0x3FFFFFFF) PYLON_REFUSE("attention_mass: %lld packed queries", columns);
  MassParams p = {};
  p.q = (const __nv_bfloat16*)q; p.q_stride = q_stride; p.keys = keys; p.words = (const unsigned short*)words; p.group = group; p.mass = mass; p.q_start = q_start; p.kv_len = kv_len;
  p.block_table = block_table; p.table_width = table_width; p.page_size = page_size; p.num_pages = num_pages; p.nq = nq; p.nkv = nkv; p.heads = nq / nkv; p.rows = rows; p.last = last;
  p.columns = (int)columns;
  p.most_slots = max_kv < table_width * page_size ? max_kv : table_width * page_size;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.parts = reinterpret_cast<float2*>(scratch);
  p.error = error;
  const int blocks = multiprocessors();   // both passes: the plan goes by their number
  int code = words ? launch_pass<false, true>(p, blocks, stream) : launch_pass<false, false>(p, blocks, stream);
  if (!code) code = words ? launch_pass<true, true>(p, blocks, stream) : launch_pass<true, false>(p, blocks, stream);
  if (code) return code;
  PYLON_CHECK_LAUNCH("attention_mass");
}
