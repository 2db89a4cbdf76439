// Attention of one or a few query rows per sequence over the paged cache (bf16 or e4m3 pages, head_dim 64 or 128).
//
//   o[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = scale * log2(e) * <q[t, h], k_j>
//
// over the keys j that row t may see, in one pass with the running maximum m. Every key and value is needed once by all query
// heads of its kv head and by all rows of its sequence, so these G * rows columns are taken together and the kernel is bound by
// streaming the cache: 2 D or 4 D bytes a key and head against G * rows * 4 D operations.
//
// Split. The sequences' lengths are on the device and differ, so the work is cut there: the list of (sequence, kv head, block of 64
// keys or more) is laid end to end and every CTA takes an equal stretch of it, whatever lengths it crosses. A (sequence, kv head)
// that falls into one stretch is finished there; one that is cut leaves a partial (O, m, l) per stretch in the workspace, which the
// second kernel joins in order. The launch depends on no length, so it can be captured.
//
// A warp streams its own tiles of keys through a ring of its own in shared memory (16-byte asynchronous copies, zero-filled where a
// sequence has no key, so that nothing stale can reach a sum), without a barrier: warps only meet at the end of a stretch's
// (sequence, kv head). Products are mma.m16n8k16 with fp32 sums, keys (for S^T = K Q^T) or head dimensions (for O^T = V^T P^T) in
// the 16 rows, query columns in the 8: at eight columns a 128-row tensor-memory tile would take the same stream through shared
// memory twice (as codes and as expanded operands), and the products are far from being the bound. Contraction order is free, so a
// thread loads 16 bytes of a row and uses them as they lie; V^T needs pairs of keys side by side, which two byte permutations per
// four bytes give.
//
// 8 bits: e4m3 becomes f16 exactly. A query column is scaled by a power of two to at most 2^14 (f16 then holds every element down
// to 2^-28 of the largest exactly), the scores come back with that, the scale of the page and the softmax scale in one factor.
// The values' scale 2^e goes into the weight, w = 2^(s + e - M) with M the running maximum of s + e, and out of it in the sum of
// weights, l = sum w 2^-e, in 32 bits: so w is at most 1 whatever the pages' scales (2^4 with a
// reference that only moves when a score passes it by that), and goes into the product as w 2^11, where f16 has 25 binary orders of
// full precision below 1 and ten more of less. bf16 pages: w = 2^(s - M) in bf16, as the rows of a bf16 product must be.
#include "paged.cuh"

namespace sb {

struct PagedAttnParams {
  PagedBatch batch;
  const __nv_bfloat16* q;
  long q_ld, q_head;                // elements between rows, between heads
  __nv_bfloat16* o;
  long o_ld, o_head;
  const uint8_t *k, *v;
  long k_page, k_head, v_page, v_head;     // bytes
  const float *ks, *vs;
  long ks_ld, vs_ld;
  int Hq, Hkv, G;
  int causal, window;               // window < 0: none
  float scale_log2;
  int zero_tail;
  float* part;                      // partials: [2 * CTAs][columns][D] of O, then [2 * CTAs][columns][2] of (m, l)
  int ctas;
  unsigned int* err;
};

#ifndef PD_CTAS
#define PD_CTAS 2
#endif
constexpr int PD_WARPS = 4, PD_STAGE = 8192, PD_START = 2;
template <int D, bool FP8> struct PagedDecode {
  static constexpr int ROW = FP8 ? D : 2 * D;                 // bytes of a key
  static constexpr int KT = PD_STAGE / 2 / ROW;               // keys of a warp's tile: 16, 32 or 64
  static constexpr int UNIT = PD_WARPS * KT;                  // keys of a block of work
  static constexpr int MT = KT / 16;                          // m-tiles of 16 keys
  static constexpr int CPR = ROW / 16;                        // 16-byte chunks of a row
  static constexpr int EPC = FP8 ? 16 : 8;                    // elements of a chunk
  static constexpr int LOADS = CPR / 4;                       // chunks of a key row that a thread takes for S
};

// Keys that any row of the sequence may see, and the units they fall into.
struct PagedSpan {
  int row0, rows, len;              // rows: at most max_rows
  int extra;                        // rows beyond that (the caller promised that there are none)
  int lo, hi;                       // [lo, hi)
  int u0, units;
};
template <int UNIT>
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnParams& p, int b) {
  const PagedSeq s = paged_seq(p.batch, b);
  PagedSpan r;
  r.row0 = s.row0;
  r.rows = min(s.rows, p.batch.max_rows);
  r.extra = s.rows - r.rows;
  r.len = s.len;
  r.lo = r.hi = r.u0 = r.units = 0;
  if (s.rows > 0) {
    if (s.len >= 0) {
      const long cap = min(static_cast<long>(p.batch.P) << p.batch.page_shift, 0x7fffff00L);
      r.hi = static_cast<int>(min(static_cast<long>(s.len) + s.rows, cap));
      if (p.window >= 0) r.lo = min(max(s.len - p.window, 0), r.hi);
    }
    r.u0 = r.lo / UNIT;
    r.units = max((r.hi + UNIT - 1) / UNIT - r.u0, 1);         // (a sequence without keys still has its rows written)
  }
  return r;
}

// The list that is cut into stretches: every (sequence, kv head) counts as its units and PD_START more for its beginning and end.
template <int UNIT>
__device__ __forceinline__ int paged_length(const PagedAttnParams& p, int b) {
  const int u = paged_span<UNIT>(p, b).units;
  return u > 0 ? (u + PD_START) * p.Hkv : 0;
}
template <int UNIT>
__device__ __forceinline__ int paged_total(const PagedAttnParams& p, int lane) {
  int n = 0;
  for (int b = lane; b < p.batch.B; b += 32) n += paged_length<UNIT>(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// The sequence that place `at` of the list belongs to (B behind the end); *before: the length of those in front of it.
template <int UNIT>
__device__ __forceinline__ int paged_find(const PagedAttnParams& p, int at, int* before, int lane) {
  int sum0 = 0;
  for (int b0 = 0; b0 < p.batch.B; b0 += 32) {
    const int n = b0 + lane < p.batch.B ? paged_length<UNIT>(p, b0 + lane) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    if (at < sum0 + all) {
      const int l = __popc(__ballot_sync(0xffffffffu, sum0 + sum <= at));
      *before = sum0 + __shfl_sync(0xffffffffu, sum - n, l);
      return b0 + l;
    }
    sum0 += all;
  }
  *before = sum0;
  return p.batch.B;
}

// Stretch c of the list is [begin(c), begin(c + 1)): equal ones, the first of them longer by one where it does not divide.
struct Stretches {
  int share, more;
  __device__ __forceinline__ Stretches(int total, int ctas) : share(total / ctas), more(total % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * share + min(c, more); }
};

// Where a CTA (or a warp's copies, running ahead) is in its stretch: units [u, u_end) of (b, kh), nothing left when they are empty.
template <int UNIT>
struct PagedWalk {
  PagedSpan s;
  int b, kh, u, u_end, left;
  __device__ __forceinline__ void enter(int x) {
    const int end = min(s.units + PD_START, x + left);
    left -= end - x;
    u = max(x - PD_START, 0);
    u_end = max(end - PD_START, 0);
  }
  __device__ __forceinline__ void next(const PagedAttnParams& p) {
    u = u_end = 0;
    while (u == u_end && left > 0) {
      if (++kh == p.Hkv) {
        kh = 0;
        do {
          if (++b >= p.batch.B) { left = 0; return; }
          s = paged_span<UNIT>(p, b);
        } while (s.units == 0);
      }
      enter(0);
    }
  }
  __device__ __forceinline__ void start(const PagedAttnParams& p, int begin, int end, int lane) {
    left = end - begin;
    b = kh = u = u_end = 0;
    if (left <= 0) return;
    int before;
    b = paged_find<UNIT>(p, begin, &before, lane);
    if (b >= p.batch.B) { left = 0; return; }
    s = paged_span<UNIT>(p, b);
    kh = (begin - before) / (s.units + PD_START);
    enter((begin - before) % (s.units + PD_START));
    if (u == u_end) next(p);
  }
};

// Byte offset of 16-byte chunk c of row r in a tile, so placed that the reads of S (rows g, chunks 2t or t) and of V (rows 2t, chunk
// g) both touch every bank once.
template <int ROW>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  if (ROW == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (2 * ((r >> 1) & 3))) << 4);
  return r * ROW + (((c & ~7) | ((c ^ r) & 7)) << 4);
}

// four e4m3 codes to two pairs of f16, exact
__device__ __forceinline__ void f16x2_of(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// transposes an 8 x 8 matrix of 16-bit elements held by the warp
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// CTAs to an SM, and the stages of a warp's ring that fit beside each other then.
template <int NT> struct PagedShape { static constexpr int CTAS = NT == 1 ? PD_CTAS : 2, NS = CTAS == 2 ? 3 : 2; };
template <int D, int NT> constexpr int paged_decode_smem() {
  return PD_WARPS * PagedShape<NT>::NS * (PD_STAGE + 64) + 16 * D * 4 + 2 * PD_WARPS * 8 * NT * 2 * 4;
}

// NT column tiles of 8.
template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(PD_WARPS * 32, PagedShape<NT>::CTAS)
paged_decode_kernel(const PagedAttnParams p) {
  using C = PagedDecode<D, FP8>;
  constexpr int NS = PagedShape<NT>::NS, KT = C::KT, MT = C::MT, UNIT = C::UNIT, ROW = C::ROW, COLS = 8 * NT, MD = D / 16, KSTEPS = D / 16;
  constexpr int RB = 2 / NT;                             // warps that put their O down at a time
  constexpr float HEAD = FP8 ? 11.f : 0.f, SLACK = FP8 ? 4.f : 8.f;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (NS * PD_STAGE);
  // per stage: [4] key scales, [4] value scales, [4] page ids of the tile's groups of 16 keys, [1] whether it has all its keys
  uint8_t* meta = smem + PD_WARPS * NS * PD_STAGE + warp * (NS * 64);
  float* red_o = reinterpret_cast<float*>(smem + PD_WARPS * NS * (PD_STAGE + 64));         // [RB][COLS][D]
  float* red_ml = red_o + 16 * D;                                                          // [2][PD_WARPS][COLS][2]

  if (p.zero_tail) {
    const int t0 = paged_tail(p.batch);
    const long n = static_cast<long>(p.batch.T - t0) * p.Hq * (D / 8);
    for (long i = blockIdx.x * (PD_WARPS * 32L) + threadIdx.x; i < n; i += gridDim.x * (PD_WARPS * 32L)) {
      const long row = i / (p.Hq * (D / 8));
      const int x = static_cast<int>(i % (p.Hq * (D / 8)));
      *reinterpret_cast<uint4*>(p.o + (t0 + row) * p.o_ld + (x / (D / 8)) * p.o_head + (x % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
  }

  const Stretches cut(paged_total<UNIT>(p, lane), gridDim.x);
  PagedWalk<UNIT> cur, ahead;
  cur.start(p, cut.begin(blockIdx.x), cut.begin(blockIdx.x + 1), lane);
  ahead = cur;

  // The warp's copies of its next tile: KT rows of keys, then of values, zeros where the sequence has no key. The pages are looked up
  // one tile ahead of their copies.
  int put = 0, id[MT];
  auto look_up = [&]() {
    const int key0 = (ahead.s.u0 + ahead.u) * UNIT + warp * KT;
    const int* row = p.batch.table + ahead.b * p.batch.table_ld;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      id[m] = -2;                                                // -2: no key of the sequence; others out of range: no page
      if (ahead.u < ahead.u_end && key0 + m * 16 + 16 > ahead.s.lo && key0 + m * 16 < ahead.s.hi) id[m] = row[(key0 + m * 16) >> p.batch.page_shift];
    }
  };
  // a lane's place in a step's 512 bytes; step i is i * 512 on, with the chunk's bits turned by that of its row
  constexpr int STEPS = 16 * C::CPR / 32;                        // copies of a lane for 16 keys; those lie together in a page
  const uint32_t lane_at = tile_offset<ROW>(lane / C::CPR, lane % C::CPR);
  auto turn = [](int i) -> uint32_t { return ROW == 256 ? (2 * i & 6) << 4 : ROW == 128 ? (4 * i & 4) << 4 : 0; };
  auto fetch = [&]() {
    if (ahead.u < ahead.u_end) {
      const int key0 = (ahead.s.u0 + ahead.u) * UNIT + warp * KT, mask = (1 << p.batch.page_shift) - 1;
      const uint32_t dst = smem_u32(ring + put * PD_STAGE);
      const uint8_t *kb = p.k + ahead.kh * p.k_head, *vb = p.v + ahead.kh * p.v_head;
      bool all = key0 >= ahead.s.lo && key0 + KT <= ahead.s.hi;
#pragma unroll
      for (int m = 0; m < MT; ++m) all = all && static_cast<unsigned>(id[m]) < static_cast<unsigned>(p.batch.num_pages);
      if (all) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t off = ((key0 + m * 16) & mask) * ROW + lane * 16;
          const uint8_t *ksrc = kb + (static_cast<uint64_t>(id[m]) * p.k_page + off), *vsrc = vb + (static_cast<uint64_t>(id[m]) * p.v_page + off);
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const uint32_t at = dst + (lane_at ^ turn(i)) + m * 16 * ROW + i * 512;
            cp_async16(at, ksrc + i * 512);
            cp_async16(at + KT * ROW, vsrc + i * 512);
          }
        }
      } else {
#pragma unroll 1
        for (int m = 0; m < MT; ++m) {
          int page = -2;
#pragma unroll
          for (int j = 0; j < MT; ++j) if (j == m) page = id[j];
          const bool good = static_cast<unsigned>(page) < static_cast<unsigned>(p.batch.num_pages);
          if (!good && page != -2 && lane == 0) atomicOr(p.err, 4u);
          const long off = static_cast<long>((key0 + m * 16) & mask) * ROW + lane * 16;
          const uint8_t* ksrc = good ? kb + static_cast<uint64_t>(page) * p.k_page + off : p.k;
          const uint8_t* vsrc = good ? vb + static_cast<uint64_t>(page) * p.v_page + off : p.v;
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const int key = key0 + m * 16 + (i * 32 + lane) / C::CPR;
            const uint32_t at = dst + (lane_at ^ turn(i)) + m * 16 * ROW + i * 512;
            const bool in = good && key >= ahead.s.lo && key < ahead.s.hi;
            cp_async16_zfill(at, in ? ksrc + i * 512 : p.k, in ? 16 : 0);
            cp_async16_zfill(at + KT * ROW, in ? vsrc + i * 512 : p.v, in ? 16 : 0);
          }
        }
      }
      if (lane < MT) {
        int page = 0;
#pragma unroll
        for (int m = 0; m < MT; ++m) if (lane == m) page = id[m];
        const bool good = static_cast<unsigned>(page) < static_cast<unsigned>(p.batch.num_pages);
        uint8_t* at = meta + put * 64 + lane * 4;
        *reinterpret_cast<int*>(at + 32) = good ? page : -1;
        if (lane == 0) *reinterpret_cast<int*>(at + 48) = all ? 1 : 0;
        if (FP8) {
          cp_async4(smem_u32(at), p.ks + (good ? page * p.ks_ld + ahead.kh : 0));
          cp_async4(smem_u32(at + 16), p.vs + (good ? page * p.vs_ld + ahead.kh : 0));
        }
      }
      if (++ahead.u == ahead.u_end) ahead.next(p);
      look_up();
    }
    cp_async_commit();
    put = put + 1 == NS ? 0 : put + 1;
  };
  look_up();
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) fetch();

  int take = 0, parity = 0;
  while (cur.u < cur.u_end) {
    const PagedSpan s = cur.s;
    const int cols = s.rows * p.G;
    // ---- the query columns: operand B of S^T, in the order of the elements that a thread loads of a key
    uint32_t qf[NT][KSTEPS][2];
    float colf[NT][2];
    int clo[NT][2], chi[NT][2];              // keys that column 2t, 2t + 1 of the tile may see: [clo, chi)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = n * 8 + g;
      const __nv_bfloat16* src = p.q + (s.row0 + c / p.G) * p.q_ld + (cur.kh * p.G + c % p.G) * p.q_head;
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int chunk = C::LOADS == 1 ? t : C::LOADS == 2 ? 2 * t + j : 2 * t + (j & 1) + 8 * (j >> 1);
#pragma unroll
        for (int k = 0; k < C::EPC / 4; ++k) {
          uint2 w = make_uint2(0, 0);
          if (c < cols) w = *reinterpret_cast<const uint2*>(src + chunk * C::EPC + 4 * k);
          qf[n][j * (C::EPC / 4) + k][0] = w.x;
          qf[n][j * (C::EPC / 4) + k][1] = w.y;
        }
      }
      float back = p.scale_log2;
      if (FP8) {
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) most = fmaxf(most, fmaxf(fabsf(bf16_lo(qf[n][k][h])), fabsf(bf16_hi(qf[n][k][h]))));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100);
        if (most == 0.f || !(most < INFINITY)) e = 14;
        const float mul = exp_scale(14 - e);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) qf[n][k][h] = pack_f16(bf16_lo(qf[n][k][h]) * mul, bf16_hi(qf[n][k][h]) * mul);
        back *= exp_scale(e - 14);
      }
      colf[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);
      colf[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = n * 8 + 2 * t + h;
        const long pos = static_cast<long>(s.len) + col / p.G;
        clo[n][h] = p.window >= 0 ? static_cast<int>(max(pos - p.window, 0L)) : 0;
        chi[n][h] = s.hi;
        if (p.causal) chi[n][h] = static_cast<int>(min(static_cast<long>(s.hi), pos + 1));
        else if (p.window >= 0) chi[n][h] = static_cast<int>(min(static_cast<long>(s.hi), pos + p.window + 1));
        if (col >= cols) chi[n][h] = 0;
      }
    }
    // keys that every column sees
    const int all_lo = p.window >= 0 ? static_cast<int>(max(static_cast<long>(s.len) + s.rows - 1 - p.window, 0L)) : 0;
    const int all_hi = p.causal ? static_cast<int>(min(static_cast<long>(s.hi), s.len + 1L))
                                : p.window >= 0 ? static_cast<int>(min(static_cast<long>(s.hi), s.len + p.window + 1L)) : s.hi;

    float acc[NT][MD][4], M[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d = 0; d < MD; ++d) acc[n][d][0] = acc[n][d][1] = acc[n][d][2] = acc[n][d][3] = 0.f;
      M[n][0] = M[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

#pragma unroll 1
    for (int u = cur.u; u < cur.u_end; ++u) {
      cp_async_wait_group<NS - 2>();
      __syncwarp();                            // the tile is there; and every lane is done with the one before it
      fetch();
      const uint8_t* tile = ring + take * PD_STAGE;
      const uint8_t* mt_meta = meta + take * 64;
      take = take + 1 == NS ? 0 : take + 1;
      const int key0 = (s.u0 + u) * UNIT + warp * KT;
      if (key0 >= s.hi || key0 + KT <= s.lo) continue;
      // ---- S^T
      float sc[NT][MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][m][0] = sc[n][m][1] = sc[n][m][2] = sc[n][m][3] = 0.f;
#pragma unroll
        for (int j = 0; j < C::LOADS; ++j) {
          const int chunk = C::LOADS == 1 ? t : C::LOADS == 2 ? 2 * t + j : 2 * t + (j & 1) + 8 * (j >> 1);
          const uint4 x = *reinterpret_cast<const uint4*>(tile + tile_offset<ROW>(m * 16 + g, chunk));
          const uint4 y = *reinterpret_cast<const uint4*>(tile + tile_offset<ROW>(m * 16 + g + 8, chunk));
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int k = 0; k < C::EPC / 4; ++k) {
            uint32_t a[4];
            if (FP8) {
              f16x2_of(xw[k], a[0], a[2]);
              f16x2_of(yw[k], a[1], a[3]);
            } else {
              a[0] = xw[(2 * k) & 3]; a[1] = yw[(2 * k) & 3]; a[2] = xw[(2 * k + 1) & 3]; a[3] = yw[(2 * k + 1) & 3];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<FP8>(sc[n][m], a, qf[n][j * (C::EPC / 4) + k][0], qf[n][j * (C::EPC / 4) + k][1]);
          }
        }
      }
      // ---- scores with their scales and masks; in 8 bits they are s + e from here on, e the value scale's exponent
      float vinv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float kscale = 1.f, ve = 0.f;
        vinv[m] = 1.f;
        if (FP8) {
          kscale = *reinterpret_cast<const float*>(mt_meta + m * 4);
          const int e = min(max(scale_exp(*reinterpret_cast<const float*>(mt_meta + 16 + m * 4)), PAGED_LEAST_EXP), PAGED_MOST_EXP);
          ve = static_cast<float>(e);
          vinv[m] = exp_scale(-e);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = FP8 ? colf[n][h] * kscale : colf[n][h];
            sc[n][m][h] = FP8 ? fmaf(sc[n][m][h], f, ve) : sc[n][m][h] * f;
            sc[n][m][2 + h] = FP8 ? fmaf(sc[n][m][2 + h], f, ve) : sc[n][m][2 + h] * f;
          }
        }
      }
      if (key0 < all_lo || key0 + KT > all_hi || *reinterpret_cast<const int*>(mt_meta + 48) == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const bool there = *reinterpret_cast<const int*>(mt_meta + 32 + m * 4) >= 0;
          const int key = key0 + m * 16 + g;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!there || key < clo[n][h] || key >= chi[n][h]) sc[n][m][h] = -INFINITY;
              if (!there || key + 8 < clo[n][h] || key + 8 >= chi[n][h]) sc[n][m][2 + h] = -INFINITY;
            }
        }
      }
      // ---- running maximum (the reference only moves when a score passes it by SLACK: weights of 2^(HEAD + SLACK) at most fit f16)
      bool grow = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = -INFINITY;
#pragma unroll
          for (int m = 0; m < MT; ++m) x = fmaxf(x, fmaxf(sc[n][m][h], sc[n][m][2 + h]));
          top[n][h] = x;
          grow = grow || x > M[n][h] + SLACK;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = fmaxf(top[n][h], M[n][h]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float alpha = M[n][h] == -INFINITY ? 0.f : fast_exp2(M[n][h] - x);
            M[n][h] = x;
            l[n][h] *= alpha;
#pragma unroll
            for (int d = 0; d < MD; ++d) { acc[n][d][h] *= alpha; acc[n][d][2 + h] *= alpha; }
          }
      }
      // ---- weights, and operand B of O^T: pairs of keys of a column
      uint32_t pf[NT][MT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float r0 = (M[n][0] == -INFINITY ? 0.f : M[n][0]) - HEAD, r1 = (M[n][1] == -INFINITY ? 0.f : M[n][1]) - HEAD;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float w0 = fast_exp2(sc[n][m][0] - r0), w1 = fast_exp2(sc[n][m][1] - r1);
          const float w2 = fast_exp2(sc[n][m][2] - r0), w3 = fast_exp2(sc[n][m][3] - r1);
          l[n][0] = FP8 ? fmaf(w0 + w2, vinv[m], l[n][0]) : l[n][0] + (w0 + w2);
          l[n][1] = FP8 ? fmaf(w1 + w3, vinv[m], l[n][1]) : l[n][1] + (w1 + w3);
          pf[n][m][0] = transpose8x8(FP8 ? pack_f16(w0, w1) : pack_bf16(w0, w1));
          pf[n][m][1] = transpose8x8(FP8 ? pack_f16(w2, w3) : pack_bf16(w2, w3));
        }
      }
      // ---- O^T
      const uint8_t* vt = tile + KT * ROW;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = m * 16 + 2 * t;
        constexpr int WORDS = FP8 ? D / 32 : D / 16;         // words of a key that a thread takes: its D / 8 dimensions
        uint32_t w[4][WORDS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = r + (i & 1) + 8 * (i >> 1);
          if (WORDS == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(vt + tile_offset<ROW>(row, g >> 1) + 8 * (g & 1));
            w[i][0] = x.x; w[i][1 % WORDS] = x.y;
          } else {
#pragma unroll
            for (int h = 0; h < WORDS / 4; ++h) {
              const uint4 x = *reinterpret_cast<const uint4*>(vt + tile_offset<ROW>(row, g + 8 * h));
              w[i][(4 * h) % WORDS] = x.x; w[i][(4 * h + 1) % WORDS] = x.y; w[i][(4 * h + 2) % WORDS] = x.z; w[i][(4 * h + 3) % WORDS] = x.w;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          if (FP8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {                    // dimensions 4i + 2h, 4i + 2h + 1
              const uint32_t x = __byte_perm(w[0][i], w[1][i], h ? 0x7362 : 0x5140), y = __byte_perm(w[2][i], w[3][i], h ? 0x7362 : 0x5140);
              uint32_t a[4];
              f16x2_of(x, a[0], a[1]);
              f16x2_of(y, a[2], a[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_16816<true>(acc[n][(2 * i + h) % MD], a, pf[n][m][0], pf[n][m][1]);
            }
          } else {
            const uint32_t a[4] = {__byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[0][i], w[1][i], 0x7632),
                                   __byte_perm(w[2][i], w[3][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x7632)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<false>(acc[n][i % MD], a, pf[n][m][0], pf[n][m][1]);
          }
        }
      }
    }

    // ---- the warps' parts together
    float* ml = red_ml + parity * (PD_WARPS * COLS * 2);
    parity ^= 1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 4);
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 8);
        l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 16);
        if (g == 0) *reinterpret_cast<float2*>(ml + (warp * COLS + n * 8 + 2 * t + h) * 2) = make_float2(M[n][h], l[n][h]);
      }
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < PD_WARPS / RB; ++pass) {
      if (warp / RB == pass) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = n * 8 + 2 * t + h;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < PD_WARPS; ++w) top = fmaxf(top, ml[(w * COLS + col) * 2]);
            const float f = M[n][h] == -INFINITY ? 0.f : fast_exp2(M[n][h] - top);
            float* dst = red_o + (warp % RB * COLS + col) * D;
#pragma unroll
            for (int d = 0; d < MD; ++d) {
              const int at = C::LOADS == 4 ? 64 * (d >> 2) + 8 * g + 2 * (d & 3) : (D / 8) * g + 2 * d;
              float2 x = make_float2(acc[n][d][h] * f, acc[n][d][2 + h] * f);
              if (pass) {
                const float2 y = *reinterpret_cast<const float2*>(dst + at);
                x.x += y.x; x.y += y.y;
              }
              *reinterpret_cast<float2*>(dst + at) = x;
            }
          }
      }
      __syncthreads();
    }
    const bool whole = cur.u == 0 && cur.u_end == s.units;
    const size_t part0 = (static_cast<size_t>(blockIdx.x) * 2 + (cur.u > 0 ? 0 : 1)) * COLS;
    for (int i = threadIdx.x; i < COLS * (D / 4); i += PD_WARPS * 32) {
      const int col = i / (D / 4), d = (i % (D / 4)) * 4;
      if (col >= cols) continue;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) top = fmaxf(top, ml[(w * COLS + col) * 2]);
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        const float2 x = *reinterpret_cast<const float2*>(ml + (w * COLS + col) * 2);
        sum += x.x == -INFINITY ? 0.f : x.y * fast_exp2(x.x - top);
      }
      float4 o = *reinterpret_cast<const float4*>(red_o + col * D + d);
      if (RB == 2) {
        const float4 y = *reinterpret_cast<const float4*>(red_o + ((RB - 1) * COLS + col) * D + d);
        o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
      }
      if (whole) {
        // (a sum of nothing: no key, zeros; a NaN stays one)
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const long at = (s.row0 + col / p.G) * p.o_ld + (cur.kh * p.G + col % p.G) * p.o_head + d;
        *reinterpret_cast<uint2*>(p.o + at) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part + (part0 + col) * D + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part + static_cast<size_t>(gridDim.x) * 2 * COLS * D + (part0 + col) * 2) = make_float2(top, sum);
      }
    }
    if (s.extra > 0 && cur.u == 0) {
      if (threadIdx.x == 0) atomicOr(p.err, 4u);
      for (long i = threadIdx.x; i < static_cast<long>(s.extra) * p.G * (D / 8); i += PD_WARPS * 32) {
        const long r = i / (p.G * (D / 8));
        const int x = static_cast<int>(i % (p.G * (D / 8)));
        *reinterpret_cast<uint4*>(p.o + (s.row0 + s.rows + r) * p.o_ld + (cur.kh * p.G + x / (D / 8)) * p.o_head + (x % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
      }
    }
    cur.next(p);
  }
  cp_async_wait_all();
}

// Joins what stretches cut: block (j, column) looks at the border between stretch j and j + 1, and if it is the first one inside a
// (sequence, kv head), adds up that one's partials in order. A warp takes every eighth of them, D / 32 dimensions a lane.
constexpr int PJ_WARPS = 8;
template <int D, int UNIT, int COLS>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(const PagedAttnParams p) {
  constexpr int V = D / 32;
  __shared__ float sum_o[PJ_WARPS][D], sum_l[PJ_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.y, ctas = p.ctas, c0 = blockIdx.x;
  const Stretches cut(paged_total<UNIT>(p, lane), ctas);
  const int at = cut.begin(c0 + 1);
  int before;
  const int b = paged_find<UNIT>(p, at, &before, lane);
  // every block waits for the grid in front of it, so that what follows this one follows that one too
  if (b >= p.batch.B) { asm volatile("griddepcontrol.wait;" ::: "memory"); return; }
  const PagedSpan s = paged_span<UNIT>(p, b);
  const int length = s.units + PD_START, kh = (at - before) / length, x = (at - before) % length, first = at - x;
  if (x <= PD_START || cut.begin(c0) > first + PD_START || col >= s.rows * p.G) { asm volatile("griddepcontrol.wait;" ::: "memory"); return; }
  // Its parts are the second one of stretch c0, and the first of those behind it (none of them empty: the empty ones, where there are
  // fewer units than stretches, lie behind the end of the list).
  int n = 1;
  while (c0 + n < ctas && cut.begin(c0 + n) < first + length) ++n;
  const float* ml = p.part + static_cast<size_t>(ctas) * 2 * COLS * D;
  const auto index = [&](int i) { return (static_cast<size_t>(c0 + i) * 2 + (i == 0 ? 1 : 0)) * COLS + col; };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float top = -INFINITY, o[V] = {}, sum = 0.f;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, ml[index(i) * 2]);
  top = warp_max(top);
#pragma unroll 4
  for (int i = warp; i < n; i += PJ_WARPS) {
    const float2 w = *reinterpret_cast<const float2*>(ml + index(i) * 2);
    float y[V];
    if (V == 4) {
      const float4 z = *reinterpret_cast<const float4*>(p.part + index(i) * D + lane * V);
      y[0] = z.x; y[1] = z.y; y[2 % V] = z.z; y[3 % V] = z.w;
    } else {
      const float2 z = *reinterpret_cast<const float2*>(p.part + index(i) * D + lane * V);
      y[0] = z.x; y[1] = z.y;
    }
    const float f = w.x == -INFINITY ? 0.f : fast_exp2(w.x - top);
    sum += w.y * f;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] += y[v] * f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sum_o[warp][lane * V + v] = o[v];
  if (lane == 0) sum_l[warp] = sum;
  __syncthreads();
  if (threadIdx.x < D) {
    float a = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < PJ_WARPS; ++w) { a += sum_o[w][threadIdx.x]; l += sum_l[w]; }
    p.o[(s.row0 + col / p.G) * p.o_ld + (kh * p.G + col % p.G) * p.o_head + threadIdx.x] = __float2bfloat16(a * (l == 0.f ? 0.f : 1.f / l));
  }
}

template <int D, bool FP8, int NT>
static int launch_paged_decode(PagedAttnParams& p, cudaStream_t st) {
  using C = PagedDecode<D, FP8>;
  constexpr int smem = paged_decode_smem<D, NT>();
  static bool attr_set[64] = {false};
  int dev = 0;
  SB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    SB_CHECK_CUDA(cudaFuncSetAttribute(paged_decode_kernel<D, FP8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set[dev & 63] = true;
  }
  paged_decode_kernel<D, FP8, NT><<<p.ctas, PD_WARPS * 32, smem, st>>>(p);
  SB_CHECK_CUDA(cudaGetLastError());
  if (p.ctas > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.ctas - 1, min(8 * NT, p.batch.max_rows * p.G));
    cfg.blockDim = dim3(PJ_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    // programmatic dependent launch: before `griddepcontrol.wait` the grid reads the batch's description, which the kernel in
    // front of it reads too
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<D, C::UNIT, 8 * NT>, static_cast<const PagedAttnParams>(p)));
  }
  return SB_OK;
}

// CTAs of a call: as many as fit the GPU at a time, and no more than there can be units of work.
static int paged_decode_ctas(int B, int Hkv, long keys, int D, bool fp8, int columns) {
  const int unit = PD_WARPS * (PD_STAGE / 2 / (fp8 ? D : 2 * D));
  const long units = static_cast<long>(B) * Hkv * ((keys + unit - 1) / unit);
  return static_cast<int>(min(units, static_cast<long>(columns <= 8 ? PagedShape<1>::CTAS : PagedShape<2>::CTAS) * num_sms()));
}

}  // namespace sb

// fp32 elements of workspace that sb_paged_attention needs for `columns` = max_rows * Hq / Hkv (at most 16).
extern "C" long sb_paged_attention_workspace(int B, int Hkv, int P, int page, int D, int fp8, int columns) {
  const int ctas = sb::paged_decode_ctas(B, Hkv, static_cast<long>(P) * page, D, fp8 != 0, columns);
  return 2L * ctas * (columns <= 8 ? 8 : 16) * (D + 2);
}

// q, o bf16 `[T, Hq, D]` with strides between rows (_ld) and heads in elements; pages and their strides as in sb_paged_append. The rows
// of the call are in the cache already: row i of sequence b stands at lengths[b] + i and sees the keys j < lengths[b] + rows, with
// causal those j <= its own position, with window >= 0 those |j - position| <= window. zero_tail: rows behind the last sequence
// become zeros (otherwise they stay as they are).
extern "C" int sb_paged_attention(const void* q, const void* kp, const void* vp, const float* ks, const float* vs, void* o, float* work,
                                  const int* table, const int* lengths, const int* starts, int T, int B, int P, int Hq, int Hkv, int D,
                                  int page, int num_pages, int max_rows, int causal, int window, int zero_tail, float scale,
                                  long table_ld, long q_ld, long q_head, long o_ld, long o_head, long k_page, long k_head, long v_page,
                                  long v_head, long ks_ld, long vs_ld, cudaStream_t st) {
  using namespace sb;
  const int shift = page_shift_of(page);
  SB_CHECK_ARG((D == 64 || D == 128) && shift >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && T > 0 && B > 0 && P > 0 && num_pages > 0);
  SB_CHECK_ARG(max_rows > 0 && (starts != nullptr || (T == B && max_rows == 1)) && (ks == nullptr) == (vs == nullptr) && work != nullptr);
  SB_CHECK_ARG(max_rows <= 16 && max_rows * (Hq / Hkv) <= 16);
  // places of the list of work, at the shortest unit, in 32 bits
  SB_CHECK_ARG((static_cast<double>(P) * page / 64 + 1 + PD_START) * B * Hkv < 2e9);
  SB_CHECK_ARG(k_page >= 0 && v_page >= 0 && k_head >= 0 && v_head >= 0);
  const bool fp8 = ks != nullptr;
  const long size = fp8 ? 1 : 2;
  PagedAttnParams p;
  p.batch = PagedBatch{table, lengths, starts, table_ld, P, B, T, max_rows, shift, num_pages};
  p.q = static_cast<const __nv_bfloat16*>(q); p.q_ld = q_ld; p.q_head = q_head;
  p.o = static_cast<__nv_bfloat16*>(o); p.o_ld = o_ld; p.o_head = o_head;
  p.k = static_cast<const uint8_t*>(kp); p.v = static_cast<const uint8_t*>(vp);
  p.k_page = k_page * size; p.k_head = k_head * size; p.v_page = v_page * size; p.v_head = v_head * size;
  p.ks = ks; p.vs = vs; p.ks_ld = ks_ld; p.vs_ld = vs_ld;
  p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  p.causal = causal; p.window = window; p.scale_log2 = scale * 1.4426950408889634f;
  p.zero_tail = zero_tail; p.part = work;
  p.ctas = paged_decode_ctas(B, Hkv, static_cast<long>(P) * page, D, fp8, max_rows * p.G);
  p.err = error_word();
  if (!p.err) return SB_ERR_CUDA;
  const bool two = max_rows * p.G > 8;
#define SB_PD(DD, FF) return two ? launch_paged_decode<DD, FF, 2>(p, st) : launch_paged_decode<DD, FF, 1>(p, st)
  if (D == 64) { if (fp8) SB_PD(64, true); else SB_PD(64, false); }
  if (fp8) SB_PD(128, true);
  SB_PD(128, false);
#undef SB_PD
}
