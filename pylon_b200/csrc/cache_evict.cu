// Eviction from a paged cache: of every (request, KV head) that holds more than `keep` tokens, the `keep` that count most stay, and those of them that lie
// behind the first `keep` slots move into the slots that became free.
//
// What counts: a token is always kept while its place (its position in the request) is below keep_first or among the keep_recent newest; the others go by
// their mass, the largest first; of equal ones the lower slot stays.  A mass that is not a number counts less than any number.
//
// Kept tokens stay where they are if they can: only kept slots at or behind `keep` move (ascending) into freed slots before it (ascending).  Attention
// over keys that already carry their rotation does not ask for an order, sources and destinations do not overlap, and a request that evicts one token
// moves one row instead of closing the gap; what order is needed for - who is first, who is newest - the places tell.
//
// Two launches.  First every (request, KV head) chooses: a thread-block cluster of up to eight blocks, each with a stretch of the slots whose keys (the masses'
// bits in the order of the floats) stay in its shared memory; the keep-th largest key is found eight bits at a time from the blocks' histograms, read through
// distributed shared memory (equal digits of a warp are counted together: masses share their exponents), then the slots are numbered in order and sources and
// destinations listed.  One block of 512 threads took 310 us over 32,768 slots, its passes one after another; bound now by the cluster's barriers and by the
// chains of loads between them.  Then the rows of every tensor move, eight slots to a warp with all their loads in flight: bound by
// those loads.  32,768 slots of 8 heads of 128 to 4,096 (bfloat16 keys and values): 38 us with copies of mass and places; 32 rows of up to 2,112 to 2,048: 25.
// (A table may name 1.5 million slots to a row; from some point beyond that calls are refused.)
#include "common.cuh"

#include <cooperative_groups.h>
#include <limits.h>

namespace pylon {

constexpr int EVICT_THREADS = 512;
constexpr int EVICT_STAGED = 16 * 1024;      // masses and places of a block that are kept in shared memory between the passes; beyond, every pass reads the masses again
constexpr int EVICT_SMEM = 200 * 1024;
constexpr int EVICT_TENSORS = 8;

struct EvictMoves {
  char* data[EVICT_TENSORS];
  int row_bytes[EVICT_TENSORS];
  int unit[EVICT_TENSORS];      // bytes a lane moves at once: 16, 4, 2 or 1
  int count;
};

// Larger is kept first.  Masses as unsigned numbers in the order of the floats; always-kept slots above all of them, NaN below.
__device__ __forceinline__ unsigned evict_key(float mass, int place, int keep_first, int newest, int keep_recent) {
  if (place < keep_first || (long long)place > (long long)newest - keep_recent) return 0xFFFFFFFFu;
  if (mass != mass) return 0u;
  const unsigned bits = __float_as_uint(mass + 0.f);   // -0 counts as 0
  return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}

// What a block of a cluster tells the others.
struct EvictShared {
  int histogram[2][256];
  int newest, equal, holes, movers;
  int total[256];                    // of all blocks, for this block's own use
  int digit, before, alike;
};

// In place: counts[0 .. groups) become the sums of all counts before them; returns the sum of all.  By warp 0; the others wait at the caller's barrier.
__device__ __forceinline__ int prefix_groups(int* counts, int groups) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < groups; base += 32) {
    const int own = base + lane < groups ? counts[base + lane] : 0;
    int upto = own;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += other;
    }
    if (base + lane < groups) counts[base + lane] = before + upto - own;
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return before;
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(const float* mass, const int* places, const int* kv_len, const int* block_table, int table_width, int page_size,
                                                                     int num_pages, int nkv, int keep, int keep_first, int keep_recent, int* holes, int* movers, int room, int* counts, int* held,
                                                                     int staged_keys, int* error) {
  namespace cg = cooperative_groups;
  extern __shared__ unsigned dynamic[];
  __shared__ EvictShared shared;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dependency_wait();
  allow_dependents();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  auto sync_all = [&]() {
    if (ranks == 1) __syncthreads();
    else cluster.sync();
  };
  const int head = blockIdx.y, row = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = min(kv_len[row], table_width * page_size);
  const size_t pair = (size_t)row * nkv + head;
  if (tid == 0 && head == 0 && rank == 0) held[row] = min(kv_len[row], keep);
  if (n <= keep) {   // all blocks of the cluster
    if (tid == 0 && rank == 0) counts[pair] = 0;
    return;
  }
  const int* table = block_table + (size_t)row * table_width;
  const int stretch = ((n + ranks - 1) / ranks + 31) & ~31, begin = min(n, rank * stretch), end = min(n, begin + stretch), groups = (end - begin + 31) / 32;
  const bool in_shared = stretch <= staged_keys;
  unsigned* staged = dynamic;                                                     // [staged_keys]: masses, then keys
  int* staged_places = reinterpret_cast<int*>(dynamic + staged_keys);              // [staged_keys]
  int* group_counts = staged_places + staged_keys;                                 // [3][groups]: equal, holes, movers; the host's bound on groups
  const int most_groups = (((table_width * page_size + ranks - 1) / ranks + 31) & ~31) / 32;
  int* group_equal = group_counts;
  int* group_holes = group_counts + most_groups;
  int* group_movers = group_counts + 2 * most_groups;
  auto slot_index = [&](int j) -> long long {
    const int logical = j / page_size, page = table[logical];
    if (page < 0 || page >= num_pages) return -1;
    return ((long long)page * nkv + head) * page_size + (j - logical * page_size);
  };
  int newest = INT_MIN;
#pragma unroll 4
  for (int j = begin + tid; j < end; j += EVICT_THREADS) {
    const long long at = slot_index(j);
    const int place = at < 0 ? INT_MIN : places[at];
    if (in_shared) {
      staged[j - begin] = at < 0 ? 0x7FC00000u : __float_as_uint(mass[at]);   // a slot without a page: the last to be kept
      staged_places[j - begin] = at < 0 ? INT_MAX : place;
    }
    if (at < 0 && error) atomicExch(error, PYLON_ERROR_BAD_PAGE);
    newest = max(newest, place);
  }
  if (tid == 0) shared.newest = INT_MIN;
  if (tid < 256) shared.histogram[0][tid] = shared.histogram[1][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) newest = max(newest, __shfl_xor_sync(0xffffffffu, newest, offset));
  if (lane == 0) atomicMax(&shared.newest, newest);
  sync_all();
  newest = INT_MIN;
  for (int r = 0; r < ranks; ++r) newest = max(newest, cluster.map_shared_rank(&shared, r)->newest);
  auto compute_key = [&](int j) -> unsigned {
    const long long at = slot_index(j);
    return at < 0 ? 0u : evict_key(mass[at], places[at], keep_first, newest, keep_recent);
  };
  if (in_shared) {
#pragma unroll 4
    for (int j = begin + tid; j < end; j += EVICT_THREADS) {   // each thread's own
      const int place = staged_places[j - begin];
      staged[j - begin] = place == INT_MAX ? 0u : evict_key(__uint_as_float(staged[j - begin]), place, keep_first, newest, keep_recent);
    }
  }
  auto key_at = [&](int j) -> unsigned { return in_shared ? staged[j - begin] : compute_key(j); };

  // The keep-th largest key, eight bits at a time.
  unsigned threshold = 0, known = 0;
  int wanted = keep;   // how many of the keys that share the bits known so far are kept
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* histogram = shared.histogram[pass & 1];
    __syncthreads();   // the staged keys are there, the histogram is empty
    for (int base = begin + warp * 32; base < end; base += EVICT_THREADS) {
      const int j = base + lane;
      const unsigned key = j < end ? key_at(j) : 0u;
      const bool counts_here = j < end && (key & known) == threshold;
      const unsigned lanes = __ballot_sync(0xffffffffu, counts_here);
      if (counts_here) {
        const unsigned digit = (key >> shift) & 255u, alike = __match_any_sync(lanes, digit);
        if (lane == __ffs(alike) - 1) atomicAdd(&histogram[digit], __popc(alike));
      }
    }
    sync_all();   // all histograms are there; nobody reads the other one any more
    if (tid < 256) {
      int sum = 0;
      for (int r = 0; r < ranks; ++r) sum += cluster.map_shared_rank(&shared, r)->histogram[pass & 1][tid];
      shared.total[tid] = sum;
      shared.histogram[(pass & 1) ^ 1][tid] = 0;
    }
    __syncthreads();
    if (tid < 32) {   // lane l has the eight digits 255 - 8 l and below: the first lane whose digits reach `wanted`, then the digit
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mine[i] = shared.total[255 - 8 * tid - i];
        sum += mine[i];
      }
      int upto = sum;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (tid >= offset) upto += other;
      }
      const int before = upto - sum;
      if (before < wanted && upto >= wanted) {
        int seen = before;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (seen < wanted && seen + mine[i] >= wanted) {
            shared.digit = 255 - 8 * tid - i;
            shared.before = seen;
            shared.alike = mine[i];
          }
          seen += mine[i];
        }
      }
    }
    __syncthreads();
    threshold |= (unsigned)shared.digit << shift;
    known |= 255u << shift;
    wanted -= shared.before;
    if (shared.alike == wanted) break;   // all that share these bits are kept: the others do not matter
  }

  // In the slots' order, 32 to a group: who stays (of the keys whose known bits equal the threshold the first `wanted`), which slots before `keep` become free, which kept
  // ones behind it move.
  for (int group = warp; group < groups; group += EVICT_THREADS / 32) {
    const int j = begin + group * 32 + lane;
    const unsigned equal = __ballot_sync(0xffffffffu, j < end && (key_at(j) & known) == threshold);
    if (lane == 0) group_equal[group] = __popc(equal);
  }
  __syncthreads();
  if (warp == 0) {
    const int sum = prefix_groups(group_equal, groups);
    if (lane == 0) shared.equal = sum;
  }
  sync_all();
  int equal_before = 0;
  for (int r = 0; r < rank; ++r) equal_before += cluster.map_shared_rank(&shared, r)->equal;
  auto choice = [&](int group, unsigned& hole, unsigned& mover) {
    const int j = begin + group * 32 + lane;
    const unsigned key = j < end ? key_at(j) & known : 0u;
    const bool is_equal = j < end && key == threshold;
    const unsigned equal = __ballot_sync(0xffffffffu, is_equal);
    const bool kept = j < end && (key > threshold || (is_equal && equal_before + group_equal[group] + __popc(equal & ((1u << lane) - 1u)) < wanted));
    hole = __ballot_sync(0xffffffffu, j < end && j < keep && !kept);
    mover = __ballot_sync(0xffffffffu, kept && j >= keep);
  };
  for (int group = warp; group < groups; group += EVICT_THREADS / 32) {
    unsigned hole, mover;
    choice(group, hole, mover);
    if (lane == 0) {
      group_holes[group] = __popc(hole);
      group_movers[group] = __popc(mover);
    }
  }
  __syncthreads();
  if (warp == 0) {
    const int hole_sum = prefix_groups(group_holes, groups), mover_sum = prefix_groups(group_movers, groups);
    if (lane == 0) {
      shared.holes = hole_sum;
      shared.movers = mover_sum;
    }
  }
  sync_all();
  int holes_before = 0, movers_before = 0, all_holes = 0, all_movers = 0;
  for (int r = 0; r < ranks; ++r) {
    const EvictShared* other = cluster.map_shared_rank(&shared, r);
    const int other_holes = other->holes, other_movers = other->movers;
    if (r < rank) {
      holes_before += other_holes;
      movers_before += other_movers;
    }
    all_holes += other_holes;
    all_movers += other_movers;
  }
  const int most = min(room, n - keep);   // neither list can be longer (room: min(keep, slots of a row's table), and n > keep here)
  for (int group = warp; group < groups; group += EVICT_THREADS / 32) {
    unsigned hole, mover;
    choice(group, hole, mover);
    const unsigned below = (1u << lane) - 1u;
    const int j = begin + group * 32 + lane, hole_at = holes_before + group_holes[group] + __popc(hole & below), mover_at = movers_before + group_movers[group] + __popc(mover & below);
    if ((hole >> lane) & 1u && hole_at < most) holes[pair * room + hole_at] = j;
    if ((mover >> lane) & 1u && mover_at < most) movers[pair * room + mover_at] = j;
  }
  if (tid == 0 && rank == 0) counts[pair] = min(min(all_holes, all_movers), most);   // equal: keep slots stay, of which all_holes had to come from behind
  sync_all();   // nobody leaves while another block still reads its shared memory
}

// A lane's piece of a moved slot.
struct EvictPiece {
  char* data;
  int row_bytes, offset, unit;   // unit 0: none
};
__device__ __forceinline__ EvictPiece evict_piece(const EvictMoves& moves, int number) {
  for (int t = 0; t < moves.count; ++t) {
    const int pieces = moves.row_bytes[t] / moves.unit[t];
    if (number < pieces) return {moves.data[t], moves.row_bytes[t], number * moves.unit[t], moves.unit[t]};
    number -= pieces;
  }
  return {nullptr, 0, 0, 0};
}
constexpr int MOVE_SLOTS = 8;
template <typename U>
__device__ __forceinline__ void move_piece(const EvictPiece& p, const long long (&from)[MOVE_SLOTS], const long long (&to)[MOVE_SLOTS]) {
  U v[MOVE_SLOTS];
#pragma unroll
  for (int i = 0; i < MOVE_SLOTS; ++i) {
    if (to[i] >= 0) v[i] = *reinterpret_cast<const U*>(p.data + from[i] * p.row_bytes + p.offset);
  }
#pragma unroll
  for (int i = 0; i < MOVE_SLOTS; ++i) {
    if (to[i] >= 0) *reinterpret_cast<U*>(p.data + to[i] * p.row_bytes + p.offset) = v[i];
  }
}
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictMoves moves, const int* holes, const int* movers, const int* counts, const int* block_table, int table_width, int page_size,
                                                         int num_pages, int nkv, int room) {
  grid_dependency_wait();
  allow_dependents();
  const int head = blockIdx.y, row = blockIdx.z, lane = threadIdx.x & 31;
  const size_t pair = (size_t)row * nkv + head;
  const int count = counts[pair];
  const int* table = block_table + (size_t)row * table_width;
  const EvictPiece mine_first = evict_piece(moves, lane);
  int pieces = 0;
  for (int t = 0; t < moves.count; ++t) pieces += moves.row_bytes[t] / moves.unit[t];
  for (int base = (blockIdx.x * 8 + (threadIdx.x >> 5)) * MOVE_SLOTS; base < count; base += gridDim.x * 8 * MOVE_SLOTS) {
    // Lanes 0 to 7 look up where the slots come from, lanes 8 to 15 where they go.
    long long at = -1;
    const int mine = base + (lane & (MOVE_SLOTS - 1));
    if (lane < 2 * MOVE_SLOTS && mine < count) {
      const int slot = (lane < MOVE_SLOTS ? movers : holes)[pair * room + mine], logical = slot / page_size, page = table[logical];
      if (page >= 0 && page < num_pages) at = ((long long)page * nkv + head) * page_size + (slot - logical * page_size);   // others were reported by the choice
    }
    long long from[MOVE_SLOTS], to[MOVE_SLOTS];
#pragma unroll
    for (int i = 0; i < MOVE_SLOTS; ++i) {
      from[i] = __shfl_sync(0xffffffffu, at, i);
      to[i] = __shfl_sync(0xffffffffu, at, MOVE_SLOTS + i);
      if (from[i] < 0) to[i] = -1;
    }
    for (int number = lane; number < pieces; number += 32) {
      const EvictPiece piece = number == lane ? mine_first : evict_piece(moves, number);
      if (piece.unit == 16) move_piece<uint4>(piece, from, to);
      else if (piece.unit == 4) move_piece<unsigned>(piece, from, to);
      else if (piece.unit == 2) move_piece<unsigned short>(piece, from, to);
      else if (piece.unit == 1) move_piece<unsigned char>(piece, from, to);
    }
  }
}

}  // namespace pylon

using namespace pylon;

// data / row_bytes: `tensors` page tensors [num_pages, nkv, page_size, row bytes], mass and places among them; lists: int32 [rows * nkv * (2 room + 1)], room at
// least min(keep, table_width * page_size).
extern "C" int pylon_evict_slots(const float* mass, const int* places, const int* kv_len, const int* block_table, int table_width, int page_size, int num_pages, int nkv, int rows,
                                 int max_kv, int keep, int keep_first, int keep_recent, void* const* data, const int* row_bytes, int tensors, int* lists, int room, int* held, int* error,
                                 cudaStream_t stream) {
  if (rows == 0) return 0;
  if (nkv < 1 || nkv > 65535 || rows > 65535 || page_size < 1 || table_width < 1 || num_pages < 1) PYLON_REFUSE("evict_slots: %d rows, %d KV heads, page size %d", rows, nkv, page_size);
  if ((long long)table_width * page_size > 0x7FFFFFFF) PYLON_REFUSE("evict_slots: %d pages of %d slots to a row", table_width, page_size);
  if (keep < 1 || keep_first < 0 || keep_recent < 0 || keep_first > keep - keep_recent) PYLON_REFUSE("evict_slots: keep %d, of them the first %d and the newest %d", keep, keep_first, keep_recent);
  if (tensors < 1 || tensors > EVICT_TENSORS) PYLON_REFUSE("evict_slots: %d tensors: 1 to %d", tensors, EVICT_TENSORS);
  if (room < keep && room < table_width * page_size) PYLON_REFUSE("evict_slots: lists of %d slots for %d kept of %d", room, keep, table_width * page_size);
  EvictMoves moves = {};
  for (const int unit : {16, 4, 2, 1}) {   // pieces of a size side by side: lanes of a warp take the same way
    for (int t = 0; t < tensors; ++t) {
      if (row_bytes[t] < 1) PYLON_REFUSE("evict_slots: rows of %d bytes", row_bytes[t]);
      const unsigned long long low = (uintptr_t)data[t] | (unsigned)row_bytes[t];
      if ((low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1) != unit) continue;
      moves.data[moves.count] = (char*)data[t];
      moves.row_bytes[moves.count] = row_bytes[t];
      moves.unit[moves.count++] = unit;
    }
  }
  // A cluster of as many blocks as leave each at most 4,096 slots and room for the numbers of all that its table could hold, up to eight; their keys in shared memory
  // as long as they fit.
  const long long slots = (long long)table_width * page_size, longest = max_kv < slots ? max_kv : slots;
  long long ranks = 1, staged, smem;
  for (;; ranks *= 2) {
    const long long stretch = ((longest + ranks - 1) / ranks + 31) & ~31ll, most_groups = (((slots + ranks - 1) / ranks + 31) & ~31ll) / 32;
    staged = stretch <= EVICT_STAGED ? stretch : 0;
    smem = (2 * staged + 3 * most_groups) * 4;
    if (ranks == 8 || ((longest + ranks - 1) / ranks <= 4096 && smem <= EVICT_SMEM)) break;
  }
  if (smem > EVICT_SMEM) PYLON_REFUSE("evict_slots: %lld slots to a row are too many", slots);
  static bool ready[MAX_DEVICES] = {};
  bool& set = ready[current_device_slot()];
  if (!set) {
    const cudaError_t err = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EVICT_SMEM);
    if (err != cudaSuccess) PYLON_REFUSE("evict_slots: %s", cudaGetErrorString(err));
    set = true;
  }
  const long long pairs = (long long)rows * nkv;
  int* holes = lists;
  int* movers = lists + pairs * room;
  int* counts = lists + 2 * pairs * room;
  launch_dependent_cluster(evict_select_kernel, dim3((unsigned)ranks, nkv, rows), dim3(EVICT_THREADS), (size_t)smem, stream, (unsigned)ranks, mass, places, kv_len, block_table, table_width, page_size, num_pages,
                           nkv, keep, keep_first, keep_recent, holes, movers, room, counts, held, (int)staged, error);
  const int most = max_kv > keep ? (max_kv - keep < keep ? max_kv - keep : keep) : 0;
  if (most > 0) {
    const long long wanted = (most + 8 * MOVE_SLOTS - 1) / (8 * MOVE_SLOTS), fill = 1 + 16ll * multiprocessors() / pairs;
    launch_dependent(evict_move_kernel, dim3((unsigned)(wanted < fill ? wanted : fill), nkv, rows), dim3(256), 0, stream, moves, (const int*)holes, (const int*)movers, (const int*)counts,
                     block_table, table_width, page_size, num_pages, nkv, room);
  }
  PYLON_CHECK_LAUNCH("evict_slots");
}
