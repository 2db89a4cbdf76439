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
//   segments  a block per (sequence, page, head) for more rows in 8 bits: the page's rows stay in registers (in 32 bits, rotated)
//             between the maximum and the conversion, so they are read once.
#include "paged.cuh"

namespace sb {

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

// Norm and rotation of the 8 elements from `part * 8` of a head; the head's other elements are in the D / 8 lanes of the group.
template <int D>
__device__ __forceinline__ void norm_rotate(float* v, const AppendParams& p, const float* gamma, long pos, int part) {
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
    const float4 c = *reinterpret_cast<const float4*>(p.cos_t + pos * (D / 2) + part * 4);
    const float4 s = *reinterpret_cast<const float4*>(p.sin_t + pos * (D / 2) + part * 4);
    const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * cc[i] - b * sn[i];
      v[2 * i + 1] = a * sn[i] + b * cc[i];
    }
  }
}

// The largest finite magnitude of 8 values; anything infinite becomes NaN on the way, which is how a page holds it.
__device__ __forceinline__ float finite_max(float* v) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    if (!(a < INFINITY)) v[i] = __uint_as_float(0x7fffffffu);
    else m = fmaxf(m, a);
  }
  return m;
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
template <int D, bool FP8>
__global__ void __launch_bounds__(256) paged_append_rows_kernel(const AppendParams p) {
  constexpr int TPH = D / 8;
  asm volatile("griddepcontrol.launch_dependents;");
  const int heads = p.Hq + 2 * p.Hkv;
  const long item = (blockIdx.x * 256L + threadIdx.x) / TPH;
  const int part = threadIdx.x % TPH;
  const bool there = item < static_cast<long>(p.batch.T) * heads;
  const int t = there ? static_cast<int>(item / heads) : 0, h = there ? static_cast<int>(item % heads) : 0;
  // the row's sequence: the last one that starts at or before it
  int b = t;
  const bool tail = t >= paged_tail(p.batch);
  if (p.batch.starts != nullptr) {
    int lo = 0, hi = p.batch.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.batch.starts[mid] <= t) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  const PagedSeq s = paged_seq(p.batch, b);
  const bool mine = there && !tail && t >= s.row0 && t < s.row0 + s.rows;
  long pos = 0;
  int page = -1;
  if (mine && s.len >= 0) {
    pos = static_cast<long>(s.len) + (t - s.row0);
    page = pos < p.max_pos ? paged_page(p.batch, b, pos) : -1;
    if (page < 0 && h == 0 && part == 0) atomicOr(p.err, 4u);
  }
  const bool live = page >= 0;
  float v[8];
  uint4 w = make_uint4(0, 0, 0, 0);
  if (live) w = *reinterpret_cast<const uint4*>(p.qkv + t * p.ld + static_cast<long>(h) * D + part * 8);
  unpack8(w, v);
  const bool is_v = h >= p.Hq + p.Hkv;
  // (every lane of the warp takes part in the group sums; what a lane of no item computes goes nowhere)
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = v[i];
  norm_rotate<D>(u, p, h < p.Hq ? p.q_gamma : p.k_gamma, pos, part);
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = u[i];
  }
  if (h < p.Hq) {
    if (there && (mine || p.zero_tail))
      *reinterpret_cast<uint4*>(p.q + t * p.q_ld + static_cast<long>(h) * D + part * 8) = live ? pack8(v) : make_uint4(0, 0, 0, 0);
    if (!FP8) return;
  }
  const int hk = is_v ? h - p.Hq - p.Hkv : h - p.Hq;
  const int slot = static_cast<int>(pos & ((1 << p.batch.page_shift) - 1));
  if (!FP8) {
    if (live) {
      __nv_bfloat16* dst = is_v ? static_cast<__nv_bfloat16*>(p.vp) + page * p.v_page + hk * p.v_head
                                : static_cast<__nv_bfloat16*>(p.kp) + page * p.k_page + hk * p.k_head;
      *reinterpret_cast<uint4*>(dst + static_cast<long>(slot) * D + part * 8) = is_v ? w : pack8(v);
    }
    return;
  }
  float most = finite_max(v);
#pragma unroll
  for (int o = TPH / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o, TPH));
  const bool put = live && h >= p.Hq;
  float* sp = put ? (is_v ? p.vs + page * p.vs_ld + hk : p.ks + page * p.ks_ld + hk) : nullptr;
  float ratio = 1.f;
  int e = 0;
  if (put) e = grown_exp(slot > 0 ? *sp : 0.f, slot, most, &ratio);
  __syncwarp();                                        // every lane has read the old scale
  if (!put) return;
  uint8_t* dst = is_v ? static_cast<uint8_t*>(p.vp) + page * p.v_page + hk * p.v_head
                      : static_cast<uint8_t*>(p.kp) + page * p.k_page + hk * p.k_head;
  if (ratio != 1.f) move_codes(dst, slot * D, ratio, part, TPH);
  if (part == 0) *sp = exp_scale(e);
  *reinterpret_cast<uint2*>(dst + static_cast<long>(slot) * D + part * 8) = encode8(v, exp_scale(-e));
}

// ---------------------------------------------------------------- segments
// Block (x, y): the x-th (sequence, page) that gets rows, head y of the Hq + 2 Hkv. NP passes of 256 threads cover a page.
template <int D, int NP>
__global__ void __launch_bounds__(256) paged_append_segments_kernel(const AppendParams p) {
  constexpr int TPH = D / 8, RPP = 256 / TPH;        // threads of a row, rows of a pass
  __shared__ float red[8];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = p.batch.page_shift, page_rows = 1 << shift;
  // every warp finds the segment by itself: segments of 32 sequences at a time, summed over the lanes
  int seg = blockIdx.x, b = -1;
  for (int b0 = 0; b0 < p.batch.B && b < 0; b0 += 32) {
    int n = 0;
    if (b0 + lane < p.batch.B) {
      const PagedSeq s = paged_seq(p.batch, b0 + lane);
      // (a slot that is not in use has its rows zeroed, a page's worth at a time, as if it began at position 0)
      const long first = max(s.len, 0);
      if (s.rows > 0) n = static_cast<int>(((first + s.rows - 1) >> shift) - (first >> shift)) + 1;
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
      seg -= __shfl_sync(0xffffffffu, sum - n, l);
    } else {
      seg -= all;
    }
  }
  const int h = blockIdx.y;
  if (b < 0) {
    // behind the last segment: rows of no sequence, a page's worth per block
    const long t0 = paged_tail(p.batch) + static_cast<long>(seg) * page_rows;
    if (p.zero_tail && h < p.Hq)
      for (int r = threadIdx.x / TPH; r < page_rows && t0 + r < p.batch.T; r += RPP)
        *reinterpret_cast<uint4*>(p.q + (t0 + r) * p.q_ld + static_cast<long>(h) * D + (threadIdx.x % TPH) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const PagedSeq s = paged_seq(p.batch, b);
  const long first = max(s.len, 0);
  const long page_no = (first >> shift) + seg, pos0 = max(first, page_no << shift);
  const int slot0 = static_cast<int>(pos0 - (page_no << shift));
  const int n = static_cast<int>(min(first + s.rows, (page_no + 1) << shift) - pos0);
  const long row0 = s.row0 + (pos0 - first);
  int page = -1, live = 0;                             // rows of the segment that have a place: a page, and a row of the tables
  if (s.len >= 0) {
    page = paged_page(p.batch, b, pos0);
    live = page < 0 ? 0 : static_cast<int>(min(static_cast<long>(n), max(p.max_pos - pos0, 0L)));
    if (live < n && h == 0 && threadIdx.x == 0) atomicOr(p.err, 4u);
  }
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
  const float* gamma = is_q ? p.q_gamma : is_v ? nullptr : p.k_gamma;
  const int part = threadIdx.x % TPH;
  float v[NP][8], most = 0.f;
  uint4 w[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPP + threadIdx.x / TPH;
    w[i] = r < live ? *reinterpret_cast<const uint4*>(p.qkv + (row0 + r) * p.ld + static_cast<long>(h) * D + part * 8) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPP + threadIdx.x / TPH;
    unpack8(w[i], v[i]);
    if (!is_v) norm_rotate<D>(v[i], p, gamma, r < live ? pos0 + r : 0, part);
    if (is_q) {
      if (r < n)
        *reinterpret_cast<uint4*>(p.q + (row0 + r) * p.q_ld + static_cast<long>(h) * D + part * 8) = r < live ? pack8(v[i]) : make_uint4(0, 0, 0, 0);
    } else if (r < live) {
      most = fmaxf(most, finite_max(v[i]));
    }
  }
  if (is_q || live == 0) return;
  most = warp_max(most);
  if (lane == 0) red[warp] = most;
  const int hk = is_v ? h - p.Hq - p.Hkv : h - p.Hq;
  float* sp = is_v ? p.vs + page * p.vs_ld + hk : p.ks + page * p.ks_ld + hk;
  const float old = slot0 > 0 ? *sp : 0.f;
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
  const int heads = p.Hq + 2 * p.Hkv;
  if (p.ks == nullptr || one_row) {
    const long blocks = (static_cast<long>(p.batch.T) * heads * (D / 8) + 255) / 256;
    SB_CHECK_ARG(blocks <= 0x7fffffffL);
    if (p.ks == nullptr) paged_append_rows_kernel<D, false><<<static_cast<int>(blocks), 256, 0, st>>>(p);
    else paged_append_rows_kernel<D, true><<<static_cast<int>(blocks), 256, 0, st>>>(p);
  } else {
    // Rows r of a sequence touch at most (r - 1) / page + 2 pages, the rows behind the last sequence rows / page + 1 blocks.
    const int page = 1 << p.batch.page_shift;
    const long blocks = p.batch.T / page + 2L * p.batch.B + 1;
    SB_CHECK_ARG(blocks <= 0x7fffffffL && heads <= 65535);
    const dim3 grid(static_cast<unsigned>(blocks), heads);
    const int np = page * (D / 8) / 256;
    if (np <= 1) paged_append_segments_kernel<D, 1><<<grid, 256, 0, st>>>(p);
    else if (np == 2) paged_append_segments_kernel<D, 2><<<grid, 256, 0, st>>>(p);
    else if (np == 4) paged_append_segments_kernel<D, 4><<<grid, 256, 0, st>>>(p);
    else paged_append_segments_kernel<D, 8><<<grid, 256, 0, st>>>(p);
  }
  SB_CHECK_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // namespace sb

// qkv bf16 `[T, (Hq + 2 Hkv) D]` (row stride ld), q out bf16 `[T, Hq, D]` (row stride q_ld). Pages bf16 (k_scale, v_scale null) or
// e4m3 `[num_pages, Hkv, page, D]`, rows of D contiguous, with the strides between pages and between heads in elements (scales: between pages). table `[B, P]` (row stride table_ld), lengths `[B]`, starts `[B + 1]` or null (row b is sequence b's). q_gamma, k_gamma
// null: no norm. cos, sin `[max_pos, D / 2]`, null: no rotation. max_rows: the most rows of one sequence (1 selects the row kernel).
extern "C" int sb_paged_append(const void* qkv, void* q, const float* q_gamma, const float* k_gamma, const float* cos_t,
                               const float* sin_t, void* kp, void* vp, float* ks, float* vs, const int* table, const int* lengths,
                               const int* starts, int T, int B, int P, int Hq, int Hkv, int D, int page, int num_pages, int max_pos,
                               int max_rows, int zero_tail, float eps, long ld, long q_ld, long table_ld, long k_page, long k_head,
                               long v_page, long v_head, long ks_ld, long vs_ld, cudaStream_t st) {
  using namespace sb;
  const int shift = page_shift_of(page);
  SB_CHECK_ARG((D == 64 || D == 128) && shift >= 0 && Hq > 0 && Hkv > 0 && T > 0 && B > 0 && P > 0 && num_pages > 0 && max_rows > 0);
  SB_CHECK_ARG(ld % 8 == 0 && q_ld % 8 == 0 && (starts != nullptr || T == B) && (ks == nullptr) == (vs == nullptr));
  SB_CHECK_ARG((cos_t == nullptr) == (sin_t == nullptr) && (q_gamma == nullptr) == (k_gamma == nullptr) && (cos_t == nullptr || max_pos > 0));
  AppendParams p;
  p.batch = PagedBatch{table, lengths, starts, table_ld, P, B, T, max_rows, shift, num_pages};
  p.qkv = static_cast<const __nv_bfloat16*>(qkv); p.ld = ld;
  p.q = static_cast<__nv_bfloat16*>(q); p.q_ld = q_ld;
  p.q_gamma = q_gamma; p.k_gamma = k_gamma; p.eps = eps;
  p.cos_t = cos_t; p.sin_t = sin_t; p.max_pos = cos_t != nullptr ? max_pos : 0x7fffffff;
  p.kp = kp; p.vp = vp; p.ks = ks; p.vs = vs;
  p.k_page = k_page; p.k_head = k_head; p.v_page = v_page; p.v_head = v_head;
  p.ks_ld = ks_ld; p.vs_ld = vs_ld;
  p.Hq = Hq; p.Hkv = Hkv; p.zero_tail = zero_tail;
  p.err = error_word();
  if (!p.err) return SB_ERR_CUDA;
  return D == 64 ? launch_append<64>(p, starts == nullptr, st) : launch_append<128>(p, starts == nullptr, st);
}
