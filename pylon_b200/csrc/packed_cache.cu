// Pages that hold keys and values in 4 bits: the write into them (with the norm of q and k and the rotation in front of it), and back.
//
// Format of a row of d channels, in groups of G (32, 64 or 128):
//   lo = min(0, min x), hi = max(0, max x) over the group
//   step = the least number of four significant bits that is not below (hi - lo) / 15
//   zero = rint(-lo / step), code = clamp(rint(x / step) + zero, 0, 15), value = step * (code - zero)
// Since (hi - lo) / step <= 15, clamping costs at most the half step that rounding costs anyway: |value - x| <= step / 2.  |code - zero| <= 15 has four
// bits and step has four, so a value is exactly a bfloat16 (8 bits): whoever unpacks rows for another kernel loses nothing.  A group's 16-bit word is
// step as a bfloat16, whose lowest four mantissa bits are zero and hold `zero` instead: 4 + 16 / G bits an element.  A group with an element that is
// not finite, or a range that is not, has the word 0x7FC0: its step is NaN, and so are its values.  Steps below 2^-100 count as none (value 0).
// Quotients, not products with 1 / step: bfloat16 inputs hit halves exactly and often, and a product would round them either way.
//
// All of it, and the norm and the rotation in front of it, is 32-bit arithmetic in which every operation is rounded by itself (no contracted multiply-adds) and the
// order of the one sum, the norm's, is fixed: codes are whole numbers, and next to a border between two of them the last bit of a key decides.  So the pages are what the
// same formulas in elementary 32-bit operations give, bit for bit; of the formulas in 64 bits they miss one code in some ten
// million, by one, and more rarely the last bit of a group's step.  The sum of a row's d squares:
// over 64 channels the upper half of what is left is added to the lower until one is left; over others each four channels in their order first, then the
// halves of those.  (The orders of torch's mean over 64 and over 128 channels on this device, so that a statement in torch operations meets the same bits.)
#include "common.cuh"

namespace pylon {

constexpr unsigned STEP_NAN = 0x7FC0u;

// The group's word from its range; `step` as used for the quotients (infinite where there is none: every quotient is 0 then).
__device__ __forceinline__ unsigned group_word(float lo, float hi, bool bad, float& step) {
  lo = fminf(lo, 0.f);
  hi = fmaxf(hi, 0.f);
  unsigned bits = (__float_as_uint(__fdiv_rn(hi - lo, 15.f)) + 0x000FFFFFu) & 0xFFF00000u;   // up to four significant bits
  if (bad || bits >= 0x7F800000u) {
    step = INFINITY;
    return STEP_NAN;
  }
  if (bits < 0x0D800000u) {   // 2^-100
    step = INFINITY;
    return 0u;
  }
  step = __uint_as_float(bits);
  return (bits >> 16) | (unsigned)(int)rintf(__fdiv_rn(-lo, step));
}

__device__ __forceinline__ float code_value(unsigned code, unsigned word) {
  return __uint_as_float((word & 0xFFF0u) << 16) * (float)((int)code - (int)(word & 15u));
}

// Eight channels as they are loaded, and as floats.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
};
__device__ __forceinline__ void load_raw(const float* p, Raw8<float>& raw) {
  raw.a = reinterpret_cast<const float4*>(p)[0];
  raw.b = reinterpret_cast<const float4*>(p)[1];
}
__device__ __forceinline__ void load_raw(const __nv_bfloat16* p, Raw8<__nv_bfloat16>& raw) { raw.a = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void raw_floats(const Raw8<float>& raw, float (&x)[8]) {
  x[0] = raw.a.x; x[1] = raw.a.y; x[2] = raw.a.z; x[3] = raw.a.w; x[4] = raw.b.x; x[5] = raw.b.y; x[6] = raw.b.z; x[7] = raw.b.w;
}
__device__ __forceinline__ void raw_floats(const Raw8<__nv_bfloat16>& raw, float (&x)[8]) {
  const unsigned w[4] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  Raw8<T> raw;
  load_raw(p, raw);
  raw_floats(raw, x);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const unsigned*>(&pair);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The physical page of a slot, or -1 (outside the table, or a page the pool does not have).
__device__ __forceinline__ int page_of(const int* block_table, int table_width, int num_pages, int row, int slot, int page_size) {
  if (slot < 0) return -1;
  const int logical = slot / page_size;
  if (logical >= table_width) return -1;
  const int page = block_table[(size_t)row * table_width + logical];
  return page >= 0 && page < num_pages ? page : -1;
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------
// One (token, head) row to LANES lanes of a warp, eight channels to a lane: a 16-byte load of bfloat16, a 32-bit store of eight codes, and every
// reduction (norm, a group's range) a few shuffles.  (Not const __restrict__ for what the kernel ahead writes: reads through the non-coherent path may be
// moved ahead of the wait for it.)  2,036 tokens of 32 / 8 heads of 128: 21 us (its 44 MB would take 7), issue slots 64 % busy, warps waiting for fixed latencies and for
// loads; single tokens 3 us, a chain of dependent loads (row, slot, page).
template <typename T, typename Q, bool PACKED, int LANES>
__global__ void __launch_bounds__(128, 6) slot_write_kernel(
    const T* qkv, int parts, long long part_stride, Q* q_out, const float* __restrict__ q_weight, const float* __restrict__ k_weight, float eps,
    const float* __restrict__ cos_table, const float* __restrict__ sin_table, int rotary_dim, int table_positions, const int* positions, const int* slots, const int* token_row,
    const int* block_table, int table_width, int page_size, void* k_pages, void* k_words, void* v_pages, void* v_words, int* places, int num_pages, int nq, int nkv, int d, int group,
    int* error) {
  grid_dependency_wait();
  allow_dependents();
  const int lane = threadIdx.x & 31, part = lane & (LANES - 1);
  const int heads = nq + 2 * nkv, c0 = part * 8;
  const float inverse_d = 1.f / (float)d;
  const int t = blockIdx.x, position = positions[t], row = token_row[t], slot = slots[t];
  // The halves of the first rotary_dim channels: partners are rotary_dim / 16 lanes apart.  Angles are the same for all of a token's heads.
  const int half = rotary_dim >> 1;
  const bool first = c0 < half, rotates = c0 < rotary_dim;
  const int from = rotates ? (first ? lane + (half >> 3) : lane - (half >> 3)) : lane;
  const int step_heads = gridDim.y * (128 / LANES);
  int number = blockIdx.y * (128 / LANES) + threadIdx.x / LANES;
  const T* src = qkv + (size_t)t * heads * d + c0;
  Raw8<T> next = {};
  if (number < heads && c0 < d) load_raw(src + (size_t)number * d, next);
  float c[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (rotates) {
    const int p = min(max(position, 0), table_positions - 1);   // the caller checks the range
    load8<float>(cos_table + (size_t)p * half + (first ? c0 : c0 - half), c);
    load8<float>(sin_table + (size_t)p * half + (first ? c0 : c0 - half), s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = first ? -s[i] : s[i];
  }
  int page = -1, at = 0;
  if (row >= 0) {   // row < 0: a padding token, which belongs to no request
    page = page_of(block_table, table_width, num_pages, row, slot, page_size);
    if (page >= 0) at = slot % page_size;
  }
  const int last_first = blockIdx.y * (128 / LANES) + (threadIdx.x >> 5) * (32 / LANES);   // the warp's first row: all its lanes make the same turns
  for (int warp_first = last_first; warp_first < heads; warp_first += step_heads, number += step_heads) {
    const int head = min(number, heads - 1);
    const bool there = number < heads, mine = there && c0 < d;   // lanes without a row still take part in the shuffles
    const bool is_q = head < nq, is_v = head >= nq + nkv, is_k = !is_q && !is_v;
    const bool keeps = __any_sync(0xffffffffu, there && !is_q), turns = rotary_dim > 0 && __any_sync(0xffffffffu, !is_v);
    const float* weight = is_v ? nullptr : (is_q ? q_weight : k_weight);
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (mine && weight) load8<float>(weight + c0, w);
    float x[8];
    raw_floats(next, x);
    if (number + step_heads < heads && c0 < d) load_raw(src + (size_t)(number + step_heads) * d, next);   // the next row on its way
    for (int p = 1; mine && p < parts; ++p) {
      float y[8];
      load8<T>(src + (size_t)head * d + (size_t)p * part_stride, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += y[i];
    }
    if ((q_weight || k_weight) && __any_sync(0xffffffffu, weight != nullptr)) {
      float square[8], sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) square[i] = __fmul_rn(x[i], x[i]);
      if constexpr (LANES == 8) {   // 64 channels: halves
#pragma unroll
        for (int offset = LANES / 2; offset > 0; offset >>= 1)
#pragma unroll
          for (int i = 0; i < 8; ++i) square[i] = __fadd_rn(square[i], __shfl_xor_sync(0xffffffffu, square[i], offset));
#pragma unroll
        for (int half = 4; half > 0; half >>= 1)
#pragma unroll
          for (int i = 0; i < half; ++i) square[i] = __fadd_rn(square[i], square[i + half]);
        sum = square[0];
      } else {   // fours, then halves of those: a lane has two
        float low = square[0], high = square[4];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          low = __fadd_rn(low, square[i]);
          high = __fadd_rn(high, square[4 + i]);
        }
#pragma unroll
        for (int offset = LANES / 2; offset > 0; offset >>= 1) {
          low = __fadd_rn(low, __shfl_xor_sync(0xffffffffu, low, offset));
          high = __fadd_rn(high, __shfl_xor_sync(0xffffffffu, high, offset));
        }
        sum = __fadd_rn(low, high);
      }
      if (weight) {
        const float inverse = rsqrtf(__fadd_rn(__fmul_rn(sum, inverse_d), eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inverse), w[i]);
      }
    }
    if (turns) {
      float other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, x[i], from);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = is_v || !rotates ? x[i] : __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(other[i], s[i]));
    }
    if (mine && is_q) store8(q_out + ((size_t)t * nq + head) * d + c0, x);
    if (!keeps) continue;
    const bool writes = there && !is_q && page >= 0;
    if (there && !is_q && row >= 0 && page < 0 && part == 0 && error) atomicExch(error, PYLON_ERROR_BAD_PAGE);
    const int kv_head = is_q ? 0 : is_v ? head - nq - nkv : head - nq;
    const size_t dst = ((size_t)max(page, 0) * nkv + kv_head) * page_size + at;
    if (writes && is_k && part == 0 && places) places[dst] = position;
    if constexpr (PACKED) {
      float lo = 0.f, hi = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad = bad || !(fabsf(x[i]) < INFINITY);
      }
      const int members = group >> 3;   // lanes that share a group: a power of two, and groups start at multiples of it
      const unsigned bad_lanes = __ballot_sync(0xffffffffu, bad);
      bad = (bad_lanes >> (lane & ~(members - 1))) & (unsigned)((1ull << members) - 1);
#pragma unroll
      for (int offset = LANES / 2; offset > 0; offset >>= 1) {
        const float other_lo = __shfl_xor_sync(0xffffffffu, lo, offset), other_hi = __shfl_xor_sync(0xffffffffu, hi, offset);
        if (offset < members) {
          lo = fminf(lo, other_lo);
          hi = fmaxf(hi, other_hi);
        }
      }
      if (mine && writes) {
        float step;
        const unsigned word = group_word(lo, hi, bad, step);
        const float zero = (float)(word & 15u);
        unsigned codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float quotient = __fdiv_rn(x[i], step);
          float code = (quotient + 12582912.f) - 12582912.f;   // to the nearest whole number, ties to even, by adding what leaves no bits behind the point
          code = fminf(fmaxf(code + zero, 0.f), 15.f) + 8388608.f;   // (NaN, of a bad group, becomes 0)
          codes |= (__float_as_uint(code) & 15u) << (4 * i);
        }
        unsigned* pages = reinterpret_cast<unsigned*>(is_v ? v_pages : k_pages);
        pages[(dst * d + c0) >> 3] = codes;
        if ((lane & (members - 1)) == 0) reinterpret_cast<unsigned short*>(is_v ? v_words : k_words)[(dst * d + c0) / group] = (unsigned short)word;
      }
    } else if (mine && writes) {
      store8(reinterpret_cast<Q*>(is_v ? v_pages : k_pages) + dst * d + c0, x);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------
// The values of listed slots: a thread to eight channels of a key or value row.
template <typename Q>
__global__ void __launch_bounds__(256) read_packed_kernel(const unsigned* k_pages, const unsigned short* k_words, const unsigned* v_pages,
                                                          const unsigned short* v_words, Q* k_out, Q* v_out, const int* slots,
                                                          const int* token_row, const int* block_table, int table_width, int page_size, int num_pages, int nkv,
                                                          int d, int group, int num_tokens, int* error) {
  grid_dependency_wait();
  allow_dependents();
  const int chunks = d >> 3;
  const unsigned item = blockIdx.x * 256u + threadIdx.x;
  if (item >= (unsigned)(num_tokens * nkv * chunks)) return;
  const int pair = item / chunks, c = item - pair * chunks, t = pair / nkv, head = pair - t * nkv;
  const int row = token_row[t];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int page = -1, slot = 0;
  if (row >= 0) {
    slot = slots[t];
    page = page_of(block_table, table_width, num_pages, row, slot, page_size);
    if (page < 0 && c == 0 && error) atomicExch(error, PYLON_ERROR_BAD_PAGE);
  }
  const size_t src = ((size_t)max(page, 0) * nkv + head) * page_size + (page >= 0 ? slot % page_size : 0);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (blockIdx.y != which) continue;
    if (page >= 0) {
      const unsigned codes = (which ? v_pages : k_pages)[src * chunks + c], word = (which ? v_words : k_words)[(src * d + 8 * c) / group];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = code_value((codes >> (4 * i)) & 15u, word);
    }
    store8((which ? v_out : k_out) + (size_t)item * 8, x);
  }
}

// Rows' contexts as plain pages of `out_page` slots: row r's slot j goes to page r * out_width + j / out_page.  With a window only from the first slot that one of the
// row's tokens sees: the pages before it may be gone.  Slots from the multiple of 128 below that one, and from a row's length to the next
// multiple of 128, become zeros, so that a kernel that reads whole tiles meets no old numbers.  A kernel that multiplies masked weights of zero into whole
// tiles of values would hand a value that is not a number to tokens that do not see it; so a slot with such a value gets a key that is not one (masked
// scores are chosen away, not multiplied) and zeros in its place: who sees the slot has no number in any channel, nobody else is touched.  Bound by
// instructions (issue slots 77 % busy): contexts of 4,501 and some 3,000 slots of 8 heads of 128 in 14 us, 2.7 TB/s.
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
template <typename Q>
__global__ void __launch_bounds__(256) unpack_pages_kernel(const unsigned* k_pages, const unsigned short* k_words, const unsigned* v_pages, const unsigned short* v_words, Q* k_out,
                                                           Q* v_out, const int* q_start, const int* kv_len, int window, const int* block_table, int table_width, int page_size, int num_pages, int nkv, int d,
                                                           int group, int out_page, int out_width, int* lengths, int* error) {
  grid_dependency_wait();
  allow_dependents();
  const int chunks = d >> 3, row = blockIdx.z, head = blockIdx.y, at_once = 256 / chunks, c = threadIdx.x % chunks;   // a thread's channels are the same in every turn
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) {   // the lengths for whoever reads these pages: no longer than there is room
    lengths[row] = min(kv_len[row], out_width * out_page);
    if (kv_len[row] > out_width * out_page) atomicExch(error, PYLON_ERROR_BAD_PAGE);
  }
  if ((int)threadIdx.x >= at_once * chunks) return;
  const int length = min(kv_len[row], out_width * out_page), end = min((length + 127) & ~127, out_width * out_page);
  const int oldest = window > 0 ? max(0, length - (q_start[row + 1] - q_start[row]) - window + 1) : 0;
  for (int slot = (oldest & ~127) + blockIdx.x * at_once + threadIdx.x / chunks; slot < end; slot += gridDim.x * at_once) {
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = make_uint4(0u, 0u, 0u, 0u);
    float k32[8] = {}, v32[8] = {};
    if (slot >= oldest && slot < length) {
      const int page = page_of(block_table, table_width, num_pages, row, slot, page_size);
      if (page >= 0) {
        const size_t src = ((size_t)page * nkv + head) * page_size + slot % page_size;
        const unsigned k_codes = k_pages[src * chunks + c], v_codes = v_pages[src * chunks + c], k_word = k_words[(src * d + 8 * c) / group], v_word = v_words[(src * d + 8 * c) / group];
        if constexpr (sizeof(Q) == 4) {   // (the 32-bit attention reads what a token sees and nothing else)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            k32[i] = code_value((k_codes >> (4 * i)) & 15u, k_word);
            v32[i] = code_value((v_codes >> (4 * i)) & 15u, v_word);
          }
        } else {
          k = unpack8(k_codes, k_word);
          if ((v_word & 0x7F80u) != 0x7F80u) v = unpack8(v_codes, v_word);
          if (c == 0) {
            for (int w = 0; w < d / group; ++w) {
              if ((v_words[src * (d / group) + w] & 0x7F80u) == 0x7F80u) k.x = (k.x & 0xFFFF0000u) | STEP_NAN;
            }
          }
        }
      } else if (c == 0 && error) {
        atomicExch(error, PYLON_ERROR_BAD_PAGE);
      }
    }
    const int to = slot / out_page;
    const size_t dst = ((((size_t)row * out_width + to) * nkv + head) * out_page + (slot - to * out_page)) * d + 8 * c;
    if constexpr (sizeof(Q) == 4) {
      store8(k_out + dst, k32);
      store8(v_out + dst, v32);
    } else {
      *reinterpret_cast<uint4*>(k_out + dst) = k;
      *reinterpret_cast<uint4*>(v_out + dst) = v;
    }
  }
}

inline int check_sizes(const char* name, int nkv, int d, int group, int page_size, int table_width, int num_pages) {
  if (d < 32 || d > 256 || d % 8) PYLON_REFUSE("%s: head size %d: a multiple of 8 from 32 to 256 is needed", name, d);
  if ((group != 32 && group != 64 && group != 128) || d % group) PYLON_REFUSE("%s: groups of %d channels of %d: 32, 64 or 128 that divide the head size are needed", name, group, d);
  if (nkv < 1 || page_size < 1 || table_width < 1 || num_pages < 1) PYLON_REFUSE("%s: %d KV heads, page size %d, table width %d, %d pages", name, nkv, page_size, table_width, num_pages);
  return 0;
}

}  // namespace pylon

using namespace pylon;

extern "C" int pylon_slot_write(const void* qkv, int parts, long long part_stride, void* q_out, const float* q_weight, const float* k_weight, float eps, const float* cos_table,
                                const float* sin_table, int rotary_dim, int table_positions, const int* positions, const int* slots, const int* token_row, const int* block_table,
                                int table_width, int page_size, void* k_pages, void* k_words, void* v_pages, void* v_words, int* places, int num_pages, int nq, int nkv, int d,
                                int group, int num_tokens, int in_dtype, int out_dtype, int* error, cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  const bool packed = k_words != nullptr;
  if (int code = check_sizes("slot_write", nkv, d, packed ? group : 32, page_size, table_width, num_pages); code && packed) return code;
  if (d < 8 || d > 256 || d % 8 || nq < 1 || nkv < 1 || page_size < 1) PYLON_REFUSE("slot_write: head size %d: a multiple of 8 up to 256 is needed", d);
  if (rotary_dim < 0 || rotary_dim > d || rotary_dim % 16 || (rotary_dim && table_positions < 1)) PYLON_REFUSE("slot_write: rotation over %d of %d channels: a multiple of 16 is needed", rotary_dim, d);
  int lanes = 1;
  while (lanes * 8 < d) lanes *= 2;
  if (lanes < 4) lanes = 4;
  const int rows = 128 / lanes;   // (token, head) rows to a block
  const int most = (nq + 2 * nkv + rows - 1) / rows;
  if (most > 65535) PYLON_REFUSE("slot_write: %d / %d heads are too many", nq, nkv);
  // A block to a token, walking its heads, where tokens fill the device; else heads are spread over blocks as well.
  const int spread = (6 * multiprocessors() + num_tokens - 1) / num_tokens, blocks = spread < most ? spread : most;
#define PYLON_SLOT_WRITE(T, Q, P, L)                                                                                                                                  \
  launch_dependent(slot_write_kernel<T, Q, P, L>, dim3((unsigned)num_tokens, (unsigned)blocks), dim3(128), 0, stream, (const T*)qkv, parts, part_stride, (Q*)q_out,   \
                   q_weight, k_weight, eps, cos_table, sin_table, rotary_dim, table_positions, positions, slots, token_row, block_table, table_width, page_size,      \
                   k_pages, k_words, v_pages, v_words, places, num_pages, nq, nkv, d, group, error)
#define PYLON_SLOT_WRITE_LANES(T, Q, P)          \
  switch (lanes) {                               \
    case 4: PYLON_SLOT_WRITE(T, Q, P, 4); break; \
    case 8: PYLON_SLOT_WRITE(T, Q, P, 8); break; \
    case 16: PYLON_SLOT_WRITE(T, Q, P, 16); break; \
    default: PYLON_SLOT_WRITE(T, Q, P, 32);      \
  }
#define PYLON_SLOT_WRITE_PACKED(T, Q)   \
  if (packed) {                         \
    PYLON_SLOT_WRITE_LANES(T, Q, true)  \
  } else {                              \
    PYLON_SLOT_WRITE_LANES(T, Q, false) \
  }
  if (in_dtype == PYLON_DTYPE_BF16 && out_dtype == PYLON_DTYPE_BF16 && parts == 1) {
    PYLON_SLOT_WRITE_PACKED(__nv_bfloat16, __nv_bfloat16)
  } else if (in_dtype == PYLON_DTYPE_F32 && out_dtype == PYLON_DTYPE_BF16) {
    PYLON_SLOT_WRITE_PACKED(float, __nv_bfloat16)
  } else if (in_dtype == PYLON_DTYPE_F32 && out_dtype == PYLON_DTYPE_F32) {
    PYLON_SLOT_WRITE_PACKED(float, float)
  } else {
    PYLON_REFUSE("slot_write: dtypes %d / %d, %d parts", in_dtype, out_dtype, parts);
  }
  PYLON_CHECK_LAUNCH("slot_write");
}

extern "C" int pylon_read_packed(const void* k_pages, const void* k_words, const void* v_pages, const void* v_words, void* k_out, void* v_out, const int* slots, const int* token_row,
                                 const int* block_table, int table_width, int page_size, int num_pages, int nkv, int d, int group, int num_tokens, int out_dtype, int* error,
                                 cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  if (int code = check_sizes("read_packed", nkv, d, group, page_size, table_width, num_pages)) return code;
  const long long blocks = ((long long)num_tokens * nkv * (d / 8) + 255) / 256;
  if (blocks > 0x7FFFFF) PYLON_REFUSE("read_packed: %d tokens are too many for one launch", num_tokens);
#define PYLON_READ_PACKED(Q)                                                                                                                                              \
  launch_dependent(read_packed_kernel<Q>, dim3((unsigned)blocks, 2), dim3(256), 0, stream, (const unsigned*)k_pages, (const unsigned short*)k_words, (const unsigned*)v_pages, \
                   (const unsigned short*)v_words, (Q*)k_out, (Q*)v_out, slots, token_row, block_table, table_width, page_size, num_pages, nkv, d, group, num_tokens, error)
  if (out_dtype == PYLON_DTYPE_F32) PYLON_READ_PACKED(float);
  else if (out_dtype == PYLON_DTYPE_BF16) PYLON_READ_PACKED(__nv_bfloat16);
  else PYLON_REFUSE("read_packed: unknown dtype %d", out_dtype);
  PYLON_CHECK_LAUNCH("read_packed");
}

extern "C" int pylon_unpack_pages(const void* k_pages, const void* k_words, const void* v_pages, const void* v_words, void* k_out, void* v_out, const int* q_start, const int* kv_len, int window,
                                  const int* block_table, int table_width, int page_size, int num_pages, int nkv, int d, int group, int rows, int max_kv, int out_page, int out_width, int* lengths,
                                  int out_dtype, int* error, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (int code = check_sizes("unpack_pages", nkv, d, group, page_size, table_width, num_pages)) return code;
  if (!lengths || !error) PYLON_REFUSE("unpack_pages: room for the lengths and an error word are needed");
  if (window < 0 || out_page < 1 || out_width < 1 || max_kv < 1 || nkv > 65535 || rows > 65535) PYLON_REFUSE("unpack_pages: %d rows, %d KV heads, pages of %d, %d a row", rows, nkv, out_page, out_width);
  const int at_once = 256 / (d / 8);
  const long long wanted = ((long long)max_kv + 127 + at_once - 1) / at_once, most = 1 + 16ll * multiprocessors() / ((long long)rows * nkv);
#define PYLON_UNPACK(Q)                                                                                                                                                     \
  launch_dependent(unpack_pages_kernel<Q>, dim3((unsigned)(wanted < most ? wanted : most), nkv, rows), dim3(256), 0, stream, (const unsigned*)k_pages,                         \
                   (const unsigned short*)k_words, (const unsigned*)v_pages, (const unsigned short*)v_words, (Q*)k_out, (Q*)v_out, q_start, kv_len, window, block_table, table_width, \
                   page_size, num_pages, nkv, d, group, out_page, out_width, lengths, error)
  if (out_dtype == PYLON_DTYPE_F32) PYLON_UNPACK(float);
  else if (out_dtype == PYLON_DTYPE_BF16) PYLON_UNPACK(__nv_bfloat16);
  else PYLON_REFUSE("unpack_pages: unknown dtype %d", out_dtype);
  PYLON_CHECK_LAUNCH("unpack_pages");
}
