// Appending to the paged cache: the packed projection `[T, (Hq + 2 Hkv) D]` of a batch of sequences goes in, the queries come out
// normed (optionally) and rotated, the keys go into their pages the same way, the values as they are.
//
//   x <- x * rsqrt(mean(x^2) + eps) * gamma                 per q / k head, with gains
//   (x0, x1) <- (x0 c - x1 s, x0 s + x1 c)                  adjacent pairs, c and s of the row's position
// held in 32 bits until the one rounding of the store. In 8 bits a page and head has one scale 2^e: e is the smallest with
// max |x| <= 448 * 2^e over the rows that this call puts there; a page's first slot begins it anew, otherwise it only grows and
// the codes of the slots before are moved over. Nothing behind the last row is touched.
//
// It moves 2 bytes in and 1 or 2 out per element and computes little, so memory and, for one row a sequence, launch latency
// bound it. Two kernels:
//   rows      a group of D / 8 threads per (row, head), 16 bytes each. For bf16 pages, and in 8 bits where a sequence has one
//             row: the group's own maximum is then the call's.
//   segments  more rows in 8 bits: the queries as above; a block per (sequence, page, head) for keys and values, whose rows stay in
//             registers (in 32 bits, rotated) between the maximum and the conversion, so they are read once.
// Measured at 32 query heads and 8 kv heads of 128 (a call among others of a graph): one token of one sequence 2.4 us, of 64 sequences 2.6 us,
// which is what a launch takes; 8 prompts of 2048 rows 77 us into e4m3 and 69 into bf16 pages (4.8 and 5.9 TB/s), 7 of 130 to 2048 into
// e4m3 28 us (4.3 TB/s). The 8-bit form is bound by issue (61% of the slots): the conversions, and a maximum over every row. A single row that
// raises its page's scale waits for the codes before it: one sequence's 2.3 us become 6 in the middle of a page of 64 and 10 at its end.
#include "paged.cuh"

namespace sb {

// Heads that a group of threads takes where there are many rows, so that a row's place, cosines and sines are looked up once for them: 8
// prompts of 2048 rows take 129 us with 1, 79 with 4, 82 with 8 and 97 with 16 (e4m3; bf16 114, 69, 70, 77).
constexpr int HEADS = 4;
// Blocks of one head, beyond which they do: that many are on the GPU at a time. 512 sequences of one row (1536 blocks) take 4.5 us with one head
// and 3.3 with 4 in bf16 pages, 6.6 and 5.5 in e4m3; below, more blocks are the better use of it.
constexpr long MANY_BLOCKS = 148 * 8;

struct AppendParams {
  PagedBatch batch;
  const __nv_bfloat16* qkv;
  long ld;                          // elements between rows
  __nv_bfloat16* q;                 // [T, Hq, D], row stride q_ld
  long q_ld;
  const float *q_gamma, *k_gamma;   // null: no norm
  float eps;
  const float *cos_t, *sin_t;       // [max_pos, D / 2], null: no rotation
  int max_pos;
  void *kp, *vp;
  long k_page, k_head, v_page, v_head;     // elements between pages and between heads
  float *ks, *vs;                          // [num_pages, Hkv], row strides ks_ld / vs_ld; null: bf16 pages
  long ks_ld, vs_ld;
  int Hq, Hkv;
  int zero_tail;                    // rows behind the last sequence: 1 zeros, 0 left as they are
  unsigned int* err;
};

__device__ __forceinline__ void unpack8(uint4 w, float* v) {
  v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
  v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// Cosines and sines of a position for the 4 pairs from `part * 4` on.
template <int D>
__device__ __forceinline__ void turns(const AppendParams& p, long pos, int part, float* c, float* s) {
  if (p.cos_t == nullptr) return;
  const float4 a = *reinterpret_cast<const float4*>(p.cos_t + pos * (D / 2) + part * 4);
  const float4 b = *reinterpret_cast<const float4*>(p.sin_t + pos * (D / 2) + part * 4);
  c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
  s[0] = b.x; s[1] = b.y; s[2] = b.z; s[3] = b.w;
}

// Norm and rotation of the 8 elements from `part * 8` of a head; the head's other elements are in the D / 8 lanes of the group.
template <int D>
__device__ __forceinline__ void norm_rotate(float* v, const AppendParams& p, const float* gamma, int part, const float* c, const float* s) {
  if (gamma != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, D / 8);
    const float r = rsqrtf(ss / D + p.eps);
    const float4 g0 = *reinterpret_cast<const float4*>(gamma + part * 8), g1 = *reinterpret_cast<const float4*>(gamma + part * 8 + 4);
    v[0] *= r * g0.x; v[1] *= r * g0.y; v[2] *= r * g0.z; v[3] *= r * g0.w;
    v[4] *= r * g1.x; v[5] *= r * g1.y; v[6] *= r * g1.z; v[7] *= r * g1.w;
  }
  if (p.cos_t != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * c[i] - b * s[i];
      v[2 * i + 1] = a * s[i] + b * c[i];
    }
  }
}

// The largest finite magnitude of 8 values; anything infinite becomes NaN on the way, which is how a page holds it. (Magnitudes of floats
// are ordered as their bits are.)
__device__ __forceinline__ float finite_max(float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  if (m >= 0x7f800000u) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
      if (a >= 0x7f800000u) v[i] = __uint_as_float(0x7fffffffu);
      else m = max(m, a);
    }
  }
  return __uint_as_float(m);
}

__device__ __forceinline__ uint2 encode8(const float* v, float inv) {
  return make_uint2(e4m3x2(v[0] * inv, v[1] * inv) | (e4m3x2(v[2] * inv, v[3] * inv) << 16),
                    e4m3x2(v[4] * inv, v[5] * inv) | (e4m3x2(v[6] * inv, v[7] * inv) << 16));
}

// `bytes` (a multiple of 16) of codes from `at` on, moved to a scale that is 2^-d of what it was: thread i of n.
__device__ __forceinline__ void move_codes(uint8_t* at, int bytes, float ratio, int i, int n) {
  for (int k = i * 16; k < bytes; k += n * 16) {
    uint4 w = *reinterpret_cast<const uint4*>(at + k);
    uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = e4m3x2_to_float2(u[j] & 0xffffu), b = e4m3x2_to_float2(u[j] >> 16);
      u[j] = e4m3x2(a.x * ratio, a.y * ratio) | (e4m3x2(b.x * ratio, b.y * ratio) << 16);
    }
    *reinterpret_cast<uint4*>(at + k) = w;
  }
}

// log2 of the scale of a page and head after rows of the largest magnitude `most` went in from `slot` on, and 2^(old - new), 1 if it stays.
__device__ __forceinline__ int grown_exp(float old, int slot, float most, float* ratio) {
  int e = e4m3_exp(most);
  *ratio = 1.f;
  if (slot > 0) {
    const int o = min(max(scale_exp(old), PAGED_LEAST_EXP), PAGED_MOST_EXP);
    if (o < e) *ratio = o - e < -30 ? 0.f : exp_scale(o - e);     // 448 * 2^-30 is below half the smallest step
    else e = o;
  }
  return e;
}

// ---------------------------------------------------------------- rows
// Rows from blockIdx `bx` * 256 / (D / 8) on, one per group, and the heads from h0 on that lie below `heads`, HPT at most. The
// projection's rows are asked for before anything is known of their sequence: their addresses need nothing but the row's number.
template <int D, bool FP8, int HPT>
__device__ __forceinline__ void append_rows(const AppendParams& p, int bx, int h0, int heads) {
  constexpr int TPH = D / 8;
  const int part = threadIdx.x % TPH;
  const long row = bx * static_cast<long>(256 / TPH) + threadIdx.x / TPH;
  const bool there = row < p.batch.T;
  const int t = there ? static_cast<int>(row) : p.batch.T - 1;
  uint4 w[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (h0 + i < heads) w[i] = *reinterpret_cast<const uint4*>(p.qkv + t * p.ld + static_cast<long>(h0 + i) * D + part * 8);
  const int b = p.batch.starts != nullptr ? paged_row_seq<TPH>(p.batch, t) : t;
  const PagedSeq s = paged_seq(p.batch, b);
  const bool mine = there && t < paged_tail(p.batch) && t >= s.row0 && t < s.row0 + s.rows;
  long pos = 0;
  int page = -1;
  if (mine && s.len >= 0) {
    pos = static_cast<long>(s.len) + (t - s.row0);
    page = pos < p.max_pos ? paged_page(p.batch, b, pos) : -1;
    if (page < 0 && h0 == 0 && part == 0) atomicOr(p.err, 4u);
  }
  const bool live = page >= 0;
  const int slot = static_cast<int>(pos & ((1 << p.batch.page_shift) - 1));
  float c[4], sn[4];
  turns<D>(p, live ? pos : 0, part, c, sn);
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) return;
    const bool is_v = h >= p.Hq + p.Hkv;
    float v[8];
    unpack8(w[i], v);
    if (!is_v) norm_rotate<D>(v, p, h < p.Hq ? p.q_gamma : p.k_gamma, part, c, sn);
    if (h < p.Hq) {
      if (there && (mine || p.zero_tail))
        *reinterpret_cast<uint4*>(p.q + t * p.q_ld + static_cast<long>(h) * D + part * 8) = live ? pack8(v) : make_uint4(0, 0, 0, 0);
      continue;
    }
    const int hk = is_v ? h - p.Hq - p.Hkv : h - p.Hq;
    if (!FP8) {
      if (live) {
        __nv_bfloat16* dst = is_v ? static_cast<__nv_bfloat16*>(p.vp) + page * p.v_page + hk * p.v_head
                                  : static_cast<__nv_bfloat16*>(p.kp) + page * p.k_page + hk * p.k_head;
        *reinterpret_cast<uint4*>(dst + static_cast<long>(slot) * D + part * 8) = is_v ? w[i] : pack8(v);
      }
      continue;
    }
    float most = finite_max(v);
#pragma unroll
    for (int o = TPH / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o, TPH));
    float* sp = !live ? nullptr : is_v ? p.vs + page * p.vs_ld + hk : p.ks + page * p.ks_ld + hk;
    float ratio = 1.f;
    int e = 0;
    if (live) e = grown_exp(slot > 0 ? *sp : 0.f, slot, most, &ratio);
    __syncwarp();                                        // every lane has read the old scale
    if (live) {
      uint8_t* dst = is_v ? static_cast<uint8_t*>(p.vp) + page * p.v_page + hk * p.v_head
                          : static_cast<uint8_t*>(p.kp) + page * p.k_page + hk * p.k_head;
      if (ratio != 1.f) move_codes(dst, slot * D, ratio, part, TPH);
      if (part == 0) *sp = exp_scale(e);
      *reinterpret_cast<uint2*>(dst + static_cast<long>(slot) * D + part * 8) = encode8(v, exp_scale(-e));
    }
  }
}

template <int D, bool FP8, int HPT>
__global__ void __launch_bounds__(256) paged_append_rows_kernel(const AppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  append_rows<D, FP8, HPT>(p, blockIdx.x, blockIdx.y * HPT, p.Hq + 2 * p.Hkv);
}

// ---------------------------------------------------------------- segments
// The first `q_blocks` blocks take the queries as above. Of the others, 2 Hkv per (sequence, page) that gets rows, one for each head
// of keys and of values; NP passes of 256 threads cover the
// rows that one of them can get, of a page or of max_rows.
template <int D, int NP>
__global__ void __launch_bounds__(256, NP > 4 ? 2 : 4) paged_append_segments_kernel(const AppendParams p, const int q_blocks) {
  constexpr int TPH = D / 8, RPP = 256 / TPH;        // threads of a row, rows of a pass
  __shared__ float red[8];
  asm volatile("griddepcontrol.launch_dependents;");
  const int groups = (p.Hq + HEADS - 1) / HEADS;
  if (static_cast<int>(blockIdx.x) < q_blocks) {
    append_rows<D, false, HEADS>(p, blockIdx.x / groups, static_cast<int>(blockIdx.x % groups) * HEADS, p.Hq);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = p.batch.page_shift;
  int seg = (blockIdx.x - q_blocks) / (2 * p.Hkv), b = -1;
  const int h = (blockIdx.x - q_blocks) % (2 * p.Hkv);
  // warp 0 finds the segment: segments of 32 sequences at a time, summed over the lanes
  __shared__ int found[5];
  if (warp == 0) {
    PagedSeq s;
    for (int b0 = 0; b0 < p.batch.B && b < 0; b0 += 32) {
      int n = 0;
      s = PagedSeq{0, 0, -1};
      if (b0 + lane < p.batch.B) {
        s = paged_seq(p.batch, b0 + lane);
        if (s.rows > 0 && s.len >= 0) n = static_cast<int>(((static_cast<long>(s.len) + s.rows - 1) >> shift) - (s.len >> shift)) + 1;
      }
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const int all = __shfl_sync(0xffffffffu, sum, 31);
      if (seg < all) {
        const int l = __popc(__ballot_sync(0xffffffffu, sum <= seg));      // the first lane whose sum passes it
        b = b0 + l;
        if (lane == l) {
          found[1] = seg - (sum - n);
          found[2] = s.row0;
          found[3] = s.rows;
          found[4] = s.len;
        }
      } else {
        seg -= all;
      }
    }
    if (lane == 0) found[0] = b;
  }
  __syncthreads();
  b = found[0];
  if (b < 0) return;
  seg = found[1];
  const PagedSeq s = PagedSeq{found[2], found[3], found[4]};
  const long first = s.len, page_no = (first >> shift) + seg, pos0 = max(first, page_no << shift);
  const int slot0 = static_cast<int>(pos0 - (page_no << shift));
  const int n = static_cast<int>(min(first + s.rows, (page_no + 1) << shift) - pos0);
  const long row0 = s.row0 + (pos0 - first);
  const bool is_v = h >= p.Hkv;
  const int part = threadIdx.x % TPH, hk = is_v ? h - p.Hkv : h;
  uint4 w[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPP + threadIdx.x / TPH;
    w[i] = r < n ? *reinterpret_cast<const uint4*>(p.qkv + (row0 + r) * p.ld + static_cast<long>(p.Hq + h) * D + part * 8) : make_uint4(0, 0, 0, 0);
  }
  const int page = paged_page(p.batch, b, pos0);
  // rows of the segment that have a place: a page, and a row of the tables (the queries' blocks report those that have none)
  int live = page < 0 ? 0 : static_cast<int>(min(static_cast<long>(n), max(p.max_pos - pos0, 0L)));
  if (live > NP * RPP) {                               // more rows than max_rows says
    live = NP * RPP;
    if (threadIdx.x == 0) atomicOr(p.err, 4u);
  }
  if (live == 0) return;
  float* sp = is_v ? p.vs + page * p.vs_ld + hk : p.ks + page * p.ks_ld + hk;
  const float old = slot0 > 0 ? *sp : 0.f;
  float v[NP][8], most = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPP + threadIdx.x / TPH;
    unpack8(w[i], v[i]);
    if (!is_v) {
      float c[4], sn[4];
      turns<D>(p, r < live ? pos0 + r : 0, part, c, sn);
      norm_rotate<D>(v[i], p, p.k_gamma, part, c, sn);
    }
    if (r < live) most = fmaxf(most, finite_max(v[i]));
  }
  most = warp_max(most);
  if (lane == 0) red[warp] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) most = fmaxf(most, red[i]);
  float ratio;
  const int e = grown_exp(old, slot0, most, &ratio);
  uint8_t* dst = is_v ? static_cast<uint8_t*>(p.vp) + page * p.v_page + hk * p.v_head
                      : static_cast<uint8_t*>(p.kp) + page * p.k_page + hk * p.k_head;
  if (ratio != 1.f) move_codes(dst, slot0 * D, ratio, threadIdx.x, 256);
  if (threadIdx.x == 0) *sp = exp_scale(e);                 // (every thread read the old one before the barrier)
  const float inv = exp_scale(-e);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPP + threadIdx.x / TPH;
    if (r < live) *reinterpret_cast<uint2*>(dst + static_cast<long>(slot0 + r) * D + part * 8) = encode8(v[i], inv);
  }
}

template <int D>
static int launch_append(const AppendParams& p, bool one_row, cudaStream_t st) {
  constexpr int RPB = 256 / (D / 8);
  const int heads = p.Hq + 2 * p.Hkv;
  const long rows = (static_cast<long>(p.batch.T) + RPB - 1) / RPB;
  if (p.ks == nullptr || one_row) {
    const bool many = rows * heads > MANY_BLOCKS;
    const dim3 grid(static_cast<unsigned>(rows), many ? (heads + HEADS - 1) / HEADS : heads);
    SB_CHECK_ARG(grid.y <= 65535);
    if (p.ks == nullptr) {
      if (many) paged_append_rows_kernel<D, false, HEADS><<<grid, 256, 0, st>>>(p);
      else paged_append_rows_kernel<D, false, 1><<<grid, 256, 0, st>>>(p);
    } else {
      if (many) paged_append_rows_kernel<D, true, HEADS><<<grid, 256, 0, st>>>(p);
      else paged_append_rows_kernel<D, true, 1><<<grid, 256, 0, st>>>(p);
    }
  } else {
    // Rows r of a sequence touch at most (r - 1) / page + 2 pages.
    const int page = 1 << p.batch.page_shift;
    const long q_blocks = rows * ((p.Hq + HEADS - 1) / HEADS), blocks = q_blocks + (p.batch.T / page + 2L * p.batch.B) * 2 * p.Hkv;
    SB_CHECK_ARG(blocks <= 0x7fffffffL);
    const unsigned grid = static_cast<unsigned>(blocks);
    const int np = (min(page, p.batch.max_rows) + RPB - 1) / RPB;
    if (np <= 1) paged_append_segments_kernel<D, 1><<<grid, 256, 0, st>>>(p, static_cast<int>(q_blocks));
    else if (np == 2) paged_append_segments_kernel<D, 2><<<grid, 256, 0, st>>>(p, static_cast<int>(q_blocks));
    else if (np <= 4) paged_append_segments_kernel<D, 4><<<grid, 256, 0, st>>>(p, static_cast<int>(q_blocks));
    else if constexpr (PAGED_MAX_PAGE / RPB > 4) paged_append_segments_kernel<D, 8><<<grid, 256, 0, st>>>(p, static_cast<int>(q_blocks));
  }
  SB_CHECK_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // namespace sb

extern "C" int sb_paged_append(const sb::PagedAppendArgs* args) {
  using namespace sb;
  SB_CHECK_ARG(args != nullptr);
  const PagedAppendArgs& c = *args;
  const int shift = page_shift_of(c.page);
  SB_CHECK_ARG((c.D == 64 || c.D == 128) && shift >= 0 && c.Hq > 0 && c.Hkv > 0 && c.T > 0 && c.B > 0 && c.P > 0 && c.num_pages > 0);
  SB_CHECK_ARG(c.ld % 8 == 0 && c.q_ld % 8 == 0 && c.max_rows > 0 && (c.starts != nullptr || c.T == c.B));
  SB_CHECK_ARG((c.k_scale == nullptr) == (c.v_scale == nullptr) && (c.cos == nullptr) == (c.sin == nullptr));
  SB_CHECK_ARG(aligned16(c.qkv, c.q, c.q_gamma, c.k_gamma, c.cos, c.sin, c.k, c.v));
  SB_CHECK_ARG((c.q_gamma == nullptr) == (c.k_gamma == nullptr) && (c.cos == nullptr || c.max_pos > 0));
  AppendParams p;
  p.batch = PagedBatch{c.table, c.lengths, c.starts, c.table_ld, c.P, c.B, c.T, c.max_rows, shift, c.num_pages};
  p.qkv = static_cast<const __nv_bfloat16*>(c.qkv); p.ld = c.ld;
  p.q = static_cast<__nv_bfloat16*>(c.q); p.q_ld = c.q_ld;
  p.q_gamma = c.q_gamma; p.k_gamma = c.k_gamma; p.eps = c.eps;
  p.cos_t = c.cos; p.sin_t = c.sin; p.max_pos = c.cos != nullptr ? c.max_pos : 0x7fffffff;
  p.kp = c.k; p.vp = c.v; p.ks = c.k_scale; p.vs = c.v_scale;
  p.k_page = c.k_page; p.k_head = c.k_head; p.v_page = c.v_page; p.v_head = c.v_head;
  p.ks_ld = c.k_scale_ld; p.vs_ld = c.v_scale_ld;
  p.Hq = c.Hq; p.Hkv = c.Hkv; p.zero_tail = c.zero_tail;
  p.err = error_word();
  if (!p.err) return SB_ERR_CUDA;
  return c.D == 64 ? launch_append<64>(p, c.starts == nullptr, c.stream) : launch_append<128>(p, c.starts == nullptr, c.stream);
}
