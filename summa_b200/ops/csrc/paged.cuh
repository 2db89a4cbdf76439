// What the kernels of the paged key/value cache share: the description of a cache and of a batch, and the 8-bit element.
//
// A cache layer holds its keys and its values in pages `[num_pages, Hkv, page, D]` (the rows of one page and head lie together,
// so that a head's block of keys is one contiguous piece). In 8 bits an element is an e4m3 code times the scale of its page and
// head, a power of two: dividing by it, and moving codes to a larger one, is exact but for codes that fall below the type's
// smallest step, and an e4m3 value is as precise at any scale, so nothing is lost against a scale of full precision.
//
// Sequence b has `lengths[b]` tokens in the cache before the call (negative: a slot that is not in use) and brings the rows
// `starts[b] .. starts[b + 1]` of the call (row b without `starts`); row i of it stands at position lengths[b] + i. Position p
// lives in page table[b][p / page], slot p % page. Everything that is read on the device is taken as it may come: row ranges are
// cut to the call's rows, and a position without a valid page is reported in the error word (bit 4) and skipped.
#pragma once
#include "host_util.h"
#include "sm100.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace sb {

constexpr int PAGED_LEAST_EXP = -60, PAGED_MOST_EXP = 120;   // range of log2(scale)
constexpr int PAGED_MAX_PAGE = 128;

struct PagedBatch {
  const int* table;          // [B, P], row stride table_ld
  const int* lengths;        // [B]
  const int* starts;         // [B + 1] or null
  long table_ld;
  int P, B, T, max_rows;
  int page_shift, num_pages;
};

struct PagedSeq {
  int row0, rows;            // the rows of the call that are its own
  int len;                   // tokens in the cache before the call, < 0: not in use
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
  PagedSeq s;
  s.len = p.lengths[b];
  if (p.starts == nullptr) {
    s.row0 = b;
    s.rows = 1;
  } else {
    s.row0 = min(max(p.starts[b], 0), p.T);
    s.rows = min(max(p.starts[b + 1], s.row0), p.T) - s.row0;
  }
  return s;
}

// First row behind the last sequence.
__device__ __forceinline__ int paged_tail(const PagedBatch& p) {
  return p.starts == nullptr ? p.T : min(max(p.starts[p.B], 0), p.T);
}

// The sequence of row t: the last one that starts at or before it. The groups of N lanes of a warp ask together, each for its own
// row; a step of the search looks at 32 places at once.
template <int N>
__device__ __forceinline__ int paged_row_seq(const PagedBatch& p, int t) {
  const int lane = threadIdx.x & 31;
  int mine = 0;
#pragma unroll
  for (int g = 0; g < 32; g += N) {
    const int row = __shfl_sync(0xffffffffu, t, g);
    int lo = 0, n = p.B;
    while (n > 1) {
      const int step = (n + 31) / 32;
      const bool before = lane * step < n && p.starts[lo + lane * step] <= row;
      const int hit = max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0) * step;
      lo += hit;
      n = min(n - hit, step);
    }
    if (lane / N == g / N) mine = lo;
  }
  return mine;
}

// Page of position `pos` (>= 0) of sequence b, -1 if there is none.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, long pos) {
  const long i = pos >> p.page_shift;
  if (i >= p.P) return -1;
  const int id = p.table[b * p.table_ld + i];
  return static_cast<unsigned>(id) < static_cast<unsigned>(p.num_pages) ? id : -1;
}

// log2 of a scale, which is a power of two.
__device__ __forceinline__ int scale_exp(float s) { return static_cast<int>((__float_as_uint(s) >> 23) & 255u) - 127; }
__device__ __forceinline__ float exp_scale(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The smallest e in the range with most <= 448 * 2^e (448 = 1.75 * 2^8): from the bits of `most`, no logarithm that could round.
__device__ __forceinline__ int e4m3_exp(float most) {
  const uint32_t u = __float_as_uint(most);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, PAGED_LEAST_EXP), PAGED_MOST_EXP);
}

// With 8-bit values a sum of weights l is taken against a maximum of s + e, not of s, so where the scales of two pages lie 2^126 or more apart
// a factor 2^d that brings l to another maximum may be below what 32 bits hold while l 2^d is not. It comes as two halves (e spans 180).
// And l is held 2^PAGED_SUM times as large: under scales of 2^120 the share of a key far below the largest, which many of them make count,
// would otherwise be less than 32 bits hold.
constexpr int PAGED_SUM = 20;
__device__ __forceinline__ float exp2_half(float from, float to) { return fast_exp2(0.5f * from - 0.5f * to); }

// Two values to two e4m3 codes (the first in the low byte): nearest, ties to even, NaN for NaN. Infinities come as NaN from the
// caller: the conversion itself would make the largest finite value of them.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3);
  return __half22float2(__half2(h));
}

// The arguments of the C entry points, in the layout that the caller packs (no padding: 8-byte fields first, an even number of
// 4-byte ones behind). Strides are in elements.
struct PagedAppendArgs {
  cudaStream_t stream;
  const void* qkv;                   // bf16 [T, (Hq + 2 Hkv) D], row stride ld
  void* q;                           // bf16 [T, Hq, D], row stride q_ld
  const float *q_gamma, *k_gamma;    // [D], null: no norm
  const float *cos, *sin;            // [max_pos, D / 2], null: no rotation
  void *k, *v;                       // [num_pages, Hkv, page, D]: bf16, or e4m3 with scales; rows of D lie together
  float *k_scale, *v_scale;          // [num_pages, Hkv]
  const int *table, *lengths, *starts;   // [B, P], [B], [B + 1] or null (row b is sequence b's)
  long ld, q_ld, table_ld, k_page, k_head, v_page, v_head, k_scale_ld, v_scale_ld;
  int T, B, P, Hq, Hkv, D, page, num_pages, max_pos;
  int max_rows;                      // the most rows of one sequence
  int zero_tail;                     // rows behind the last sequence: 1 zeros, 0 left as they are
  float eps;
};
struct PagedAttentionArgs {
  cudaStream_t stream;
  const void* q;                     // bf16 [T, Hq, D]
  const void *k, *v;
  const float *k_scale, *v_scale;
  void* o;                           // as q
  float* work;                       // as many floats as the workspace function says, null for none
  const int *table, *lengths, *starts;
  long q_ld, q_head, o_ld, o_head, table_ld, k_page, k_head, v_page, v_head, k_scale_ld, v_scale_ld;
  int T, B, P, Hq, Hkv, D, page, num_pages, max_rows;
  int causal, window;                // window < 0: none
  int zero_tail;
  float scale;
  int pad;
};
static_assert(sizeof(PagedAppendArgs) == 14 * 8 + 9 * 8 + 12 * 4 && sizeof(PagedAttentionArgs) == 11 * 8 + 11 * 8 + 14 * 4, "packed by the caller");

// Host: whether all of these may be read or written 16 bytes at a time.
template <typename... P> inline bool aligned16(const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ... | 0) & 15) == 0; }

// Host: log2 of a page size, -1 if it is not one that the kernels take.
inline int page_shift_of(int page) {
  return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
}

}  // namespace sb
