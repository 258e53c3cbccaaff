// Paged causal attention over 4-bit pages (format: packed_cache.cu) in float32 arithmetic, for any head size that is a multiple of 32 up to 256: the
// 32-bit path's single tokens.
//
// One block a (token, query head), or one to each 128 keys of it whose parts a second kernel joins (the borders are multiples of 128 slots, so that the order of
// a sum does not depend on what else is in the call): one token of 32
// heads of 128 over 16,384 slots 123 us, a block to a head 1,678; 15 tokens of 6 heads of 64 over some 300 slots 14 and 25.  Eight lanes share a key: each has the channels 8 s .. 8 s + 7 of every stretch of 64 (a 32-bit word of codes is eight
// channels), a score takes three shuffles, and the sixteen groups of eight lanes walk the keys side by side with a softmax of their own; the groups are
// joined at the end through shared memory.  Bound by arithmetic and by latency, not by bytes.
#include "common.cuh"

namespace pylon {

constexpr int PLAIN_GROUPS = 16;   // groups of eight lanes to a block of 128 threads
constexpr int PLAIN_SEGMENT = 128;  // keys to a part

template <int WORDS>
__device__ __forceinline__ void plain_values(const unsigned* codes, const unsigned short* words, size_t row, int s, int d, int group, float (&x)[WORDS * 8]) {
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int c = 64 * w + 8 * s;
    if (c < d) {
      const unsigned code = codes[(row * d + c) >> 3], word = words[(row * d + c) / group];
      const float step = __uint_as_float((word & 0xFFF0u) << 16);
      const int zero = word & 15u;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * w + i] = step * (float)((int)((code >> (4 * i)) & 15u) - zero);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * w + i] = 0.f;
    }
  }
}

template <typename T, int WORDS>
__global__ void __launch_bounds__(128) attention_packed_plain_kernel(const T* q, long long q_stride, const unsigned* k_pages, const unsigned short* k_words, const unsigned* v_pages,
                                                                     const unsigned short* v_words, T* out, long long out_stride, const int* slots, const int* token_row,
                                                                     const int* block_table, int table_width, int page_size, int num_pages, int nq, int nkv, int d, int group, int window,
                                                                     float scale, float* part_values, float2* part_sums, int segments, int* error) {
  __shared__ float shared_out[PLAIN_GROUPS][WORDS * 64];
  __shared__ float shared_top[PLAIN_GROUPS], shared_total[PLAIN_GROUPS];
  grid_dependency_wait();
  allow_dependents();
  const int token = blockIdx.x, head = blockIdx.y, kv_head = head / (nq / nkv);
  const int s = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int row = token_row[token];
  if (row < 0) return;   // a padding token
  const int newest = min(slots[token], table_width * page_size - 1), oldest = window > 0 ? max(0, newest - window + 1) : 0;
  float mine[WORDS * 8], sum[WORDS * 8];
#pragma unroll
  for (int e = 0; e < WORDS * 8; ++e) {
    const int c = 64 * (e >> 3) + 8 * s + (e & 7);
    mine[e] = c < d ? to_float<T>(q[(size_t)token * q_stride + (size_t)head * d + c]) * scale : 0.f;
  }
  // Without parts one stretch; else the parts z, z + gridDim.z, ... of those that the token sees.
  for (int segment = segments ? oldest / PLAIN_SEGMENT + blockIdx.z : 0; segment <= (segments ? min(newest / PLAIN_SEGMENT, segments - 1) : 0); segment += segments ? gridDim.z : 1) {
    const int first = segments ? max(oldest, segment * PLAIN_SEGMENT) : oldest, last = segments ? min(newest, segment * PLAIN_SEGMENT + PLAIN_SEGMENT - 1) : newest;
#pragma unroll
    for (int e = 0; e < WORDS * 8; ++e) sum[e] = 0.f;
    float top = -INFINITY, total = 0.f;
    // Every group of a warp makes the same number of turns, so that the shuffles have all lanes.
    for (int base = first; base <= last; base += PLAIN_GROUPS) {
      const int j = base + g;
      int page = -1;
      if (j <= last) {
        page = block_table[(size_t)row * table_width + j / page_size];
        if (page < 0 || page >= num_pages) {
          if (s == 0 && error) atomicExch(error, PYLON_ERROR_BAD_PAGE);
          page = -1;
        }
      }
      const size_t at = ((size_t)max(page, 0) * nkv + kv_head) * page_size + (page >= 0 ? j % page_size : 0);
      float x[WORDS * 8], score = 0.f;
      plain_values<WORDS>(k_pages, k_words, at, s, d, group, x);
#pragma unroll
      for (int e = 0; e < WORDS * 8; ++e) score = fmaf(mine[e], x[e], score);
#pragma unroll
      for (int offset = 4; offset > 0; offset >>= 1) score += __shfl_xor_sync(0xffffffffu, score, offset);
      if (page < 0) continue;
      const float now = fmaxf(top, score);
      if (now == -INFINITY && score == score) continue;   // nothing has weight yet
      const float keep = expf(top - now), weight = expf(score - now);
      plain_values<WORDS>(v_pages, v_words, at, s, d, group, x);
      total = total * keep + weight;
#pragma unroll
      for (int e = 0; e < WORDS * 8; ++e) sum[e] = sum[e] * keep + weight * x[e];
      top = now;
    }
#pragma unroll
    for (int e = 0; e < WORDS * 8; ++e) shared_out[g][64 * (e >> 3) + 8 * s + (e & 7)] = sum[e];
    if (s == 0) {
      shared_top[g] = top;
      shared_total[g] = total;
    }
    __syncthreads();
    float all = -INFINITY, denominator = 0.f;
#pragma unroll
    for (int i = 0; i < PLAIN_GROUPS; ++i) all = fmaxf(all, shared_top[i]);
    float factor[PLAIN_GROUPS];
#pragma unroll
    for (int i = 0; i < PLAIN_GROUPS; ++i) {
      factor[i] = shared_total[i] == 0.f ? 0.f : expf(shared_top[i] - all);
      denominator += shared_total[i] * factor[i];
    }
    const size_t part = ((size_t)token * nq + head) * segments + segment;
    if (segments && threadIdx.x == 0) part_sums[part] = make_float2(all, denominator);
    for (int c = threadIdx.x; c < d; c += 128) {
      float value = 0.f;
#pragma unroll
      for (int i = 0; i < PLAIN_GROUPS; ++i) value += shared_out[i][c] * factor[i];
      if (segments) part_values[part * d + c] = value;
      else out[(size_t)token * out_stride + (size_t)head * d + c] = from_float<T>(denominator == 0.f ? 0.f : value / denominator);
    }
    __syncthreads();   // the groups' sums are free again
  }
}

// The parts of a (token, head) in their order, a thread to a channel.
template <typename T>
__global__ void __launch_bounds__(256) attention_packed_plain_join_kernel(const float* part_values, const float2* part_sums, T* out, long long out_stride, const int* slots,
                                                                          const int* token_row, int table_width, int page_size, int d, int window, int segments) {
  grid_dependency_wait();
  allow_dependents();
  const int token = blockIdx.x, head = blockIdx.y, c = threadIdx.x;
  if (token_row[token] < 0 || c >= d) return;
  const int newest = min(slots[token], table_width * page_size - 1), oldest = window > 0 ? max(0, newest - window + 1) : 0;
  const int first = oldest / PLAIN_SEGMENT, last = min(newest / PLAIN_SEGMENT, segments - 1);
  const size_t base = ((size_t)token * gridDim.y + head) * segments;
  float all = -INFINITY, value = 0.f, denominator = 0.f;
#pragma unroll 8
  for (int i = first; i <= last; ++i) all = fmaxf(all, part_sums[base + i].x);
#pragma unroll 8
  for (int i = first; i <= last; ++i) {
    const float2 own = part_sums[base + i];
    const float factor = own.y == 0.f ? 0.f : expf(own.x - all), v = part_values[(base + i) * d + c];
    value += v * factor;
    denominator += own.y * factor;
  }
  out[(size_t)token * out_stride + (size_t)head * d + c] = from_float<T>(denominator == 0.f ? 0.f : value / denominator);
}

}  // namespace pylon

using namespace pylon;

// slots: int32 [tokens], the slot of each token in its row: it sees the slots up to its own.  segments: 0, or the parts of 128 slots that a token can see at most
// (no slots beyond them are looked at), with scratch of tokens * nq * segments * (d + 2) floats.
extern "C" int pylon_attention_packed_plain(const void* q, long long q_stride, const void* k_pages, const void* k_words, const void* v_pages, const void* v_words, void* out,
                                            long long out_stride, const int* slots, const int* token_row, const int* block_table, int table_width, int page_size, int num_pages, int nq,
                                            int nkv, int d, int group, int window, float scale, int num_tokens, int segments, float* scratch, int dtype, int* error,
                                            cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  if (segments < 0 || (segments && !scratch)) PYLON_REFUSE("paged_attention_packed: %d parts without room for them", segments);
  if (d < 32 || d > 256 || d % 32) PYLON_REFUSE("paged_attention_packed: head size %d: a multiple of 32 up to 256 is needed", d);
  if ((group != 32 && group != 64 && group != 128) || d % group) PYLON_REFUSE("paged_attention_packed: groups of %d channels of %d", group, d);
  if (nkv < 1 || nq < 1 || nq % nkv || nq > 65535 || page_size < 1 || table_width < 1 || num_pages < 1 || window < 0)
    PYLON_REFUSE("paged_attention_packed: heads %d/%d, page size %d, table width %d, window %d", nq, nkv, page_size, table_width, window);
  if ((long long)table_width * page_size > 0x7FFFFFFF) PYLON_REFUSE("paged_attention_packed: %d pages of %d slots to a row", table_width, page_size);
  float2* part_sums = reinterpret_cast<float2*>(scratch);   // the values behind them
  float* part_values = segments ? scratch + 2 * (size_t)num_tokens * nq * segments : nullptr;
  const long long wanted = 1 + 16ll * multiprocessors() / ((long long)num_tokens * nq);   // blocks to a (token, head): as many as fill the device
  const unsigned sides = segments == 0 ? 1u : (unsigned)(wanted < segments ? wanted : segments);
#define PYLON_PACKED_PLAIN(T, W)                                                                                                                                       \
  launch_dependent(attention_packed_plain_kernel<T, W>, dim3(num_tokens, nq, sides), dim3(128), 0, stream, (const T*)q, q_stride, (const unsigned*)k_pages,                   \
                   (const unsigned short*)k_words, (const unsigned*)v_pages, (const unsigned short*)v_words, (T*)out, out_stride, slots, token_row, block_table, table_width, \
                   page_size, num_pages, nq, nkv, d, group, window, scale, part_values, part_sums, segments, error);                                                                 \
  if (segments)                                                                                                                                                        \
    launch_dependent(attention_packed_plain_join_kernel<T>, dim3(num_tokens, nq), dim3(256), 0, stream, (const float*)part_values, (const float2*)part_sums, (T*)out, out_stride, \
                     slots, token_row, table_width, page_size, d, window, segments)
#define PYLON_PACKED_PLAIN_WORDS(T)          \
  if (d <= 64) {                             \
    PYLON_PACKED_PLAIN(T, 1);                \
  } else if (d <= 128) {                     \
    PYLON_PACKED_PLAIN(T, 2);                \
  } else {                                   \
    PYLON_PACKED_PLAIN(T, 4);                \
  }
  if (dtype == PYLON_DTYPE_F32) {
    PYLON_PACKED_PLAIN_WORDS(float);
  } else if (dtype == PYLON_DTYPE_BF16) {
    PYLON_PACKED_PLAIN_WORDS(__nv_bfloat16);
  } else {
    PYLON_REFUSE("paged_attention_packed: unknown dtype %d", dtype);
  }
  PYLON_CHECK_LAUNCH("paged_attention_packed");
}
