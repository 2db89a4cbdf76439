// Attention of one or a few query rows per sequence over the paged cache (bf16 or e4m3 pages, head_dim 64 or 128).
//
//   o[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = scale * log2(e) * <q[t, h], k_j>
//
// over the keys j that row t may see, in one pass with the running maximum m. Every key and value is needed once by all query
// heads of its kv head and by all rows of its sequence, so these G * rows columns are taken together and the kernel is bound by
// streaming the cache: 2 D or 4 D bytes a key and head against G * rows * 4 D operations. More than 16 columns are taken in groups of 16,
// each an item of the list below, that stream the keys again (32 columns in e4m3: 64 sequences of 4000 tokens 194 us, 87 for 4 columns).
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
// The values' scale 2^e goes into the weight, w = 2^(s + e - M) with M the running maximum of s + e, beside a sum l of 2^(s - M) in 32
// bits: so w is at most 1 whatever the pages' scales (2^4 with a
// reference that only moves when a score passes it by that), and goes into the product as w 2^11, where f16 has 25 binary orders of
// full precision below 1 and ten more of less. bf16 pages: w = 2^(s - M) in bf16, as the rows of a bf16 product must be.
//
// Measured at 32 query heads over 8 kv heads of 128, pages from memory: 64 sequences of 37 to 8191 tokens in e4m3 43.1 us (4.8 TB/s), one of
// 100,003 40.0 us (5.1 TB/s; 6.5 over what more tokens add), 12 of up to 16,000 with a window of 4096 in bf16 36.7 us (5.1 TB/s); one of 501
// 8.1 us. Beside the stream there are some 3.5 us until the first products (the batch's description, the pages, the first tiles) and 2 to 4 of the
// second kernel. Eight warps with tiles of 16 keys, three CTAs per SM with two stages and joining by the last CTA to arrive (58 us for
// 43) were slower or no faster.
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
  int groups;                       // of up to 16 columns each, that the rows and query heads of a kv head are taken in
  int causal, window;               // window < 0: none
  float scale_log2;
  int zero_tail;
  float* part;                      // partials: [2 * CTAs] of O, then [2 * CTAs][columns][2] of (m, l)
  int ctas;
  unsigned int* err;
};

constexpr int PD_WARPS = 4, PD_STAGE = 8192, PD_NS = 3;   // a warp's ring: stages of keys and values
// What a (sequence, kv head) costs beside its keys, in units: 64 sequences of 37 to 8191 tokens take 54.8 us with 1, 45.1 with 2, 42.2 with
// 3 and 42.9 with 4.
constexpr int PD_START = 3;
// Up to so many units it is not worth a cut and the joining kernel: one sequence of 500 tokens in e4m3 (4 units) 7.9 us whole and 8.6 cut, in
// bf16 (8 units) 9.6 whole and 7.0 cut.
constexpr int PD_WHOLE = 5;
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

// How the list of (sequence, kv head) is cut: places [begin(c), begin(c + 1)) are stretch c, equal ones, the first of them longer by one
// where it does not divide. Each counts as its units and PD_START more for its beginning and end; but where all of them are short
// (PD_WHOLE units at most) each is one place, and nothing is cut.
struct Stretches {
  int share, more;
  bool whole;
  __device__ __forceinline__ int length(int units) const { return units <= 0 ? 0 : whole ? 1 : units + PD_START; }
  __device__ __forceinline__ int begin(int c) const { return c * share + min(c, more); }
  // the stretch that place x lies in
  __device__ __forceinline__ int of(int x) const {
    const int longer = more * (share + 1);
    return x < longer ? x / (share + 1) : more + (x - longer) / share;    // (share is 0 only if all places lie in the longer ones)
  }
};

// Cuts the list into `ctas` stretches and finds the sequence at the beginning of stretch c (B behind the end of the list); *at: that
// place, *before: the places in front of the sequence. By a whole warp.
template <int UNIT>
__device__ __forceinline__ int paged_locate(const PagedAttnParams& p, int c, int ctas, Stretches* cut, int* at, int* before) {
  const int lane = threadIdx.x & 31, B = p.batch.B;
  int units = lane < B ? paged_span<UNIT>(p, lane).units : 0;
  int all = units, some = units > 0, most = units;
  for (int b = lane + 32; b < B; b += 32) {
    const int u = paged_span<UNIT>(p, b).units;
    all += u; some += u > 0; most = max(most, u);
  }
  cut->whole = __reduce_max_sync(0xffffffffu, most) <= PD_WHOLE;
  const int total = __reduce_add_sync(0xffffffffu, cut->whole ? some : all + some * PD_START) * (p.Hkv * p.groups);
  cut->share = total / ctas;
  cut->more = total - cut->share * ctas;
  *at = cut->begin(c);
  int front = 0;
  for (int b0 = 0;;) {
    const int n = cut->length(units) * (p.Hkv * p.groups);
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned in_front = __ballot_sync(0xffffffffu, front + sum <= *at);
    if (in_front != 0xffffffffu) {
      const int l = __popc(in_front);
      *before = front + __shfl_sync(0xffffffffu, sum - n, l);
      return b0 + l;
    }
    front += __shfl_sync(0xffffffffu, sum, 31);
    if ((b0 += 32) >= B) break;
    units = b0 + lane < B ? paged_span<UNIT>(p, b0 + lane).units : 0;
  }
  *before = front;
  return B;
}

// Where a CTA (or a warp's copies, running ahead) is in its stretch: units [u, u_end) of (b, kh), nothing left when they are empty.
template <int UNIT>
struct PagedWalk {
  PagedSpan s;
  int b, item, u, u_end, left;      // item: kv head and group of columns
  int kh, col0;                     // of the item: its kv head, its first column
  bool whole;
  __device__ __forceinline__ void enter(int x, const PagedAttnParams& p) {
    kh = p.groups == 1 ? item : item / p.groups;
    col0 = (item - kh * p.groups) * 16;
    if (whole) { --left; u = 0; u_end = s.units; return; }
    const int end = min(s.units + PD_START, x + left);
    left -= end - x;
    u = max(x - PD_START, 0);
    u_end = max(end - PD_START, 0);
  }
  __device__ __forceinline__ void next(const PagedAttnParams& p) {
    u = u_end = 0;
    while (u == u_end && left > 0) {
      if (++item == p.Hkv * p.groups) {
        item = 0;
        do {
          if (++b >= p.batch.B) { left = 0; return; }
          s = paged_span<UNIT>(p, b);
        } while (s.units == 0);
      }
      enter(0, p);
    }
  }
  __device__ __forceinline__ void start(const PagedAttnParams& p, int c, int ctas) {
    Stretches cut;
    int at, before;
    b = paged_locate<UNIT>(p, c, ctas, &cut, &at, &before);
    left = cut.begin(c + 1) - at;
    whole = cut.whole;
    item = kh = col0 = u = u_end = 0;
    if (left <= 0 || b >= p.batch.B) { left = 0; return; }
    s = paged_span<UNIT>(p, b);
    const int length = cut.length(s.units);
    item = (at - before) / length;
    enter(at - before - item * length, p);
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

// The first of the two dimensions that accumulator quad d of a thread of group g holds.
template <int D, bool FP8>
__device__ __forceinline__ int paged_dim(int g, int d) {
  return !FP8 && D == 128 ? 64 * (d >> 2) + 8 * g + 2 * (d & 3) : (D / 8) * g + 2 * d;
}

// Shared memory: the rings; per stage 64 bytes of scales and page ids; two warps' O and all warps' (m, l) where they meet.
template <int D, int NT> constexpr int paged_decode_smem() {
  return PD_WARPS * PD_NS * (PD_STAGE + 64) + (NT == 1 ? 2 : 1) * 8 * NT * D * 4 + 2 * PD_WARPS * 8 * NT * 2 * 4;
}

// NT column tiles of 8.
template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(PD_WARPS * 32, 2)
paged_decode_kernel(const PagedAttnParams p) {
  using C = PagedDecode<D, FP8>;
  constexpr int NS = PD_NS, KT = C::KT, MT = C::MT, UNIT = C::UNIT, ROW = C::ROW, COLS = 8 * NT, MD = D / 16, KSTEPS = D / 16;
  constexpr int RB = NT == 1 ? 2 : 1;                    // warps that put their O down at a time (two CTAs have to fit an SM)
  constexpr int QUADS = NT * MD;                         // accumulators of a thread, in fours
  constexpr float HEAD = FP8 ? 11.f : 0.f, SLACK = FP8 ? 4.f : 8.f, SUM = FP8 ? PAGED_SUM : 0.f;
  extern __shared__ __align__(128) uint8_t smem[];
  // Nothing is read before the wait, and the joining kernel, which reads the batch's description before its own, starts after it.
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (NS * PD_STAGE);
  // per stage: [4] key scales, [4] value scales, [4] page ids of the tile's groups of 16 keys, [1] whether it has all its keys
  uint8_t* meta = smem + PD_WARPS * NS * PD_STAGE + warp * (NS * 64);
  float4* red_o = reinterpret_cast<float4*>(smem + PD_WARPS * NS * (PD_STAGE + 64));       // [RB][QUADS][32]
  float* red_ml = reinterpret_cast<float*>(red_o + RB * QUADS * 32);                       // [2][PD_WARPS][COLS][2]

  PagedWalk<UNIT> cur, ahead;
  cur.start(p, blockIdx.x, gridDim.x);
  ahead = cur;

  // The query columns as they lie, operand B of S^T in the order of the elements that a thread loads of a key. Those of the first (sequence,
  // kv head) are asked for before its keys.
  uint32_t qf[NT][KSTEPS][2];
  auto load_q = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = cur.col0 + n * 8 + g;
      const __nv_bfloat16* src = p.q + (cur.s.row0 + c / p.G) * p.q_ld + (cur.kh * p.G + c % p.G) * p.q_head;
      const bool there = cur.u < cur.u_end && c < cur.s.rows * p.G;
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int chunk = C::LOADS == 1 ? t : C::LOADS == 2 ? 2 * t + j : 2 * t + (j & 1) + 8 * (j >> 1);
#pragma unroll
        for (int k = 0; k < C::EPC / 8; ++k) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (there) w = *reinterpret_cast<const uint4*>(src + chunk * C::EPC + 8 * k);
          const int at = j * (C::EPC / 4) + 2 * k;
          qf[n][at][0] = w.x; qf[n][at][1] = w.y; qf[n][at + 1][0] = w.z; qf[n][at + 1][1] = w.w;
        }
      }
    }
  };
  load_q();

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
      if (__builtin_expect(all, 1)) {
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
      } else {                                         // (an edge of the sequence, or a page that is none)
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
      if (__builtin_expect(++ahead.u == ahead.u_end, 0)) ahead.next(p);
      look_up();
    }
    cp_async_commit();
    put = put + 1 == NS ? 0 : put + 1;
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) fetch();

  if (p.zero_tail) {
    const int t0 = paged_tail(p.batch);
    const long n = static_cast<long>(p.batch.T - t0) * p.Hq * (D / 8);
    for (long i = blockIdx.x * (PD_WARPS * 32L) + threadIdx.x; i < n; i += gridDim.x * (PD_WARPS * 32L)) {
      const long row = i / (p.Hq * (D / 8));
      const int x = static_cast<int>(i % (p.Hq * (D / 8)));
      *reinterpret_cast<uint4*>(p.o + (t0 + row) * p.o_ld + (x / (D / 8)) * p.o_head + (x % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
  }

  int take = 0, parity = 0;
  while (cur.u < cur.u_end) {
    const PagedSpan s = cur.s;
    const int col0 = cur.col0, cols = s.rows * p.G;
    float colf[NT][2];
    int clo[NT][2], chi[NT][2];              // keys that column 2t, 2t + 1 of the tile may see: [clo, chi)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
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
        const int col = col0 + n * 8 + 2 * t + h;
        const long pos = static_cast<long>(s.len) + col / p.G;
        clo[n][h] = p.window >= 0 ? static_cast<int>(min(max(pos - p.window, 0L), static_cast<long>(s.hi))) : 0;
        chi[n][h] = s.hi;
        if (p.causal) chi[n][h] = static_cast<int>(min(static_cast<long>(s.hi), pos + 1));
        else if (p.window >= 0) chi[n][h] = static_cast<int>(min(static_cast<long>(s.hi), pos + p.window + 1));
        if (col >= cols) chi[n][h] = 0;
      }
    }
    // keys that every column sees
    const int all_lo = p.window >= 0 ? static_cast<int>(min(max(static_cast<long>(s.len) + s.rows - 1 - p.window, 0L), static_cast<long>(s.hi))) : 0;
    const int all_hi = p.causal ? static_cast<int>(min(static_cast<long>(s.hi), s.len + 1L))
                                : p.window >= 0 ? static_cast<int>(min(static_cast<long>(s.hi), static_cast<long>(s.len) + p.window + 1)) : s.hi;

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
      float ve[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float kscale = 1.f;
        ve[m] = 0.f;
        if (FP8) {
          kscale = *reinterpret_cast<const float*>(mt_meta + m * 4);
          const int e = min(max(scale_exp(*reinterpret_cast<const float*>(mt_meta + 16 + m * 4)), PAGED_LEAST_EXP), PAGED_MOST_EXP);
          ve[m] = static_cast<float>(e);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = FP8 ? colf[n][h] * kscale : colf[n][h];
            sc[n][m][h] = FP8 ? fmaf(sc[n][m][h], f, ve[m]) : sc[n][m][h] * f;
            sc[n][m][2 + h] = FP8 ? fmaf(sc[n][m][2 + h], f, ve[m]) : sc[n][m][2 + h] * f;
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
            const float half = M[n][h] == -INFINITY ? 0.f : FP8 ? exp2_half(M[n][h], x) : fast_exp2(M[n][h] - x), alpha = FP8 ? half * half : half;
            M[n][h] = x;
            l[n][h] *= half;
            if (FP8) l[n][h] *= half;
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
          // (from the scores, not as w 2^-e: of pages 2^120 apart the one's w is nothing beside the other's, its share of l is not)
          const float q0 = r0 - SUM + ve[m], q1 = r1 - SUM + ve[m];
          l[n][0] += FP8 ? fast_exp2(sc[n][m][0] - q0) + fast_exp2(sc[n][m][2] - q0) : w0 + w2;
          l[n][1] += FP8 ? fast_exp2(sc[n][m][1] - q1) + fast_exp2(sc[n][m][3] - q1) : w1 + w3;
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
    // (O goes through shared memory and the workspace as the threads hold it: quad i of lane is dimensions at(i), at(i) + 1 of columns
    // 2t, 2t + 1 of column tile i / MD)
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = n * 8 + 2 * t + h;
        top[n][h] = -INFINITY;
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) top[n][h] = fmaxf(top[n][h], ml[(w * COLS + col) * 2]);
        const float f = M[n][h] == -INFINITY ? 0.f : fast_exp2(M[n][h] - top[n][h]);
#pragma unroll
        for (int d = 0; d < MD; ++d) { acc[n][d][h] *= f; acc[n][d][2 + h] *= f; }
      }
#pragma unroll
    for (int pass = 0; pass < PD_WARPS / RB; ++pass) {
      if (warp / RB == pass) {
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
          float4* at = red_o + (warp % RB * QUADS + i) * 32 + lane;
          const float* a = acc[i / MD][i % MD];
          float4 x = make_float4(a[0], a[1], a[2], a[3]);
          if (pass) { const float4 y = *at; x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w); }
          *at = x;
        }
      }
      __syncthreads();
    }
    const bool whole = cur.u == 0 && cur.u_end == s.units;
    const size_t part = static_cast<size_t>(blockIdx.x) * 2 + (cur.u > 0 ? 0 : 1);
    float4* part_o = reinterpret_cast<float4*>(p.part) + part * (QUADS * 32);
    float2* part_ml = reinterpret_cast<float2*>(p.part + static_cast<size_t>(gridDim.x) * 2 * COLS * D) + part * COLS;
#pragma unroll
    for (int i = warp; i < QUADS; i += PD_WARPS) {
      float4 o = red_o[i * 32 + lane];
      if (RB == 2) {
        const float4 y = red_o[((RB - 1) * QUADS + i) * 32 + lane];
        o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
      }
      if (!whole) part_o[i * 32 + lane] = o;
      const int n = i / MD;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = n * 8 + 2 * t + h;
        float tp = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) tp = fmaxf(tp, ml[(w * COLS + col) * 2]);
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) {
          const float2 x = *reinterpret_cast<const float2*>(ml + (w * COLS + col) * 2);
          if (FP8) {
            const float half = exp2_half(x.x, tp);
            sum += x.x == -INFINITY ? 0.f : x.y * half * half;
          } else {
            sum += x.x == -INFINITY ? 0.f : x.y * fast_exp2(x.x - tp);
          }
        }
        if (!whole) {
          if (i % MD == 0 && g == 0) part_ml[col] = make_float2(tp, sum);
        } else if (col0 + col < cols) {
          // (a sum of nothing: no key, zeros; a NaN stays one)
          const float inv = sum == 0.f ? 0.f : (FP8 ? 1 << PAGED_SUM : 1) / sum;
          const int c = col0 + col;
          const long to = (s.row0 + c / p.G) * p.o_ld + (cur.kh * p.G + c % p.G) * p.o_head + paged_dim<D, FP8>(g, i % MD);
          *reinterpret_cast<uint32_t*>(p.o + to) = h ? pack_bf16(o.y * inv, o.w * inv) : pack_bf16(o.x * inv, o.z * inv);
        }
      }
    }
    // rows beyond the promised ones, or positions behind the table's end
    if (__builtin_expect((s.extra > 0 || (s.len >= 0 && s.hi < static_cast<long>(s.len) + s.rows)) && cur.u == 0 && col0 == 0, 0)) {
      if (threadIdx.x == 0) atomicOr(p.err, 4u);
      for (long i = threadIdx.x; i < static_cast<long>(s.extra) * p.G * (D / 8); i += PD_WARPS * 32) {
        const long r = i / (p.G * (D / 8));
        const int x = static_cast<int>(i % (p.G * (D / 8)));
        *reinterpret_cast<uint4*>(p.o + (s.row0 + s.rows + r) * p.o_ld + (cur.kh * p.G + x / (D / 8)) * p.o_head + (x % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
      }
    }
    cur.next(p);
    load_q();
  }
  cp_async_wait_all();
}

// Joins what stretches cut: block j looks at the border between stretch j and j + 1. If it lies inside a (sequence, kv head), the blocks of
// that one's borders share its quads of O (see above), and each adds up all the partials of its own, always in the same order. Few and
// small blocks, so that most of them wait beside the kernel in front of them with their border looked up; three to an SM, since the registers
// of a fourth spilled (64 sequences of 2000 tokens in e4m3 51.9 us with four, 49.6 with three, drafts of 8 sequences 18.4 and 16.9).
constexpr int PJ_WARPS = 8, PJ_PARTS = 5;
template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(PJ_WARPS * 32, 3) paged_join_kernel(const PagedAttnParams p) {
  constexpr int COLS = 8 * NT, MD = D / 16, QUADS = NT * MD;
  __shared__ float4 sum_o[PJ_WARPS][32], sum_ml[PJ_WARPS][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, ctas = p.ctas;
  asm volatile("griddepcontrol.launch_dependents;");
  Stretches cut;
  int at, before;
  const int b = paged_locate<PagedDecode<D, FP8>::UNIT>(p, blockIdx.x + 1, ctas, &cut, &at, &before);
  PagedSpan s;
  int item = 0, n = 0, c0 = 0;
  if (!cut.whole && b < p.batch.B) {
    s = paged_span<PagedDecode<D, FP8>::UNIT>(p, b);
    const int length = cut.length(s.units);
    item = (at - before) / length;
    const int x = at - before - item * length;
    if (x > PD_START) {
      // Its parts are the second one of stretch c0, where its first unit lies, and the first one of each behind it up to that of its last.
      c0 = cut.of(at - x + PD_START);
      n = cut.of(at - x + length - 1) - c0 + 1;
    }
  }
  // every block waits for the grid in front of it, so that what follows this one follows that one too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n == 0) return;
  const float4* ml = reinterpret_cast<const float4*>(p.part + static_cast<size_t>(ctas) * 2 * COLS * D) + static_cast<size_t>(c0) * COLS;
  const float4* po = reinterpret_cast<const float4*>(p.part) + static_cast<size_t>(c0) * (2 * QUADS * 32) + lane;
  const auto index = [&](int i) { return i == 0 ? 1 : 2 * i; };
  // from one maximum to another (0: nothing there); in 8 bits in halves, which l takes one after the other
  const auto factor = [](float from, float to) { return from == -INFINITY ? 0.f : FP8 ? exp2_half(from, to) : fast_exp2(from - to); };
  const auto rest = [](float f) { return FP8 ? f : 1.f; };
  const auto whole = [](float f) { return FP8 ? f * f : f; };
  const int first = blockIdx.x - c0, step = n - 1, mine = (QUADS - first + step - 1) / step;   // quads first, first + step, ...
  // Few quads: several warps on each, a part every `split`.
  const int split = mine <= 1 ? 8 : mine <= 2 ? 4 : mine <= 4 ? 2 : 1;
  for (int k0 = 0; k0 < mine; k0 += PJ_WARPS / split) {
    const int k = k0 + warp / split, q = first + k * step, pair = q / MD * 4 + t;      // pair: columns 2t, 2t + 1 of the quad's tile
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // one round of loads for up to PJ_PARTS parts, each round's maximum with the one so far
    for (int i0 = warp % split; i0 < n && k < mine; i0 += PJ_PARTS * split) {
      float4 y[PJ_PARTS], w[PJ_PARTS];
#pragma unroll
      for (int j = 0; j < PJ_PARTS; ++j) {
        const int i = min(i0 + j * split, n - 1);
        y[j] = po[(index(i) * QUADS + q) * 32];
        w[j] = ml[index(i) * (COLS / 2) + pair];               // (m, l) of the two columns
      }
      float n0 = m0, n1 = m1;
#pragma unroll
      for (int j = 0; j < PJ_PARTS; ++j) {
        if (i0 + j * split >= n) w[j].x = w[j].z = -INFINITY;
        n0 = fmaxf(n0, w[j].x);
        n1 = fmaxf(n1, w[j].z);
      }
      const float a0 = factor(m0, n0), a1 = factor(m1, n1);
      m0 = n0; m1 = n1;
      l0 = l0 * a0 * rest(a0); o.x *= whole(a0); o.z *= whole(a0);
      l1 = l1 * a1 * rest(a1); o.y *= whole(a1); o.w *= whole(a1);
#pragma unroll
      for (int j = 0; j < PJ_PARTS; ++j) {
        if (i0 + j * split >= n) continue;
        const float f0 = factor(w[j].x, m0), f1 = factor(w[j].z, m1);
        l0 += w[j].y * f0 * rest(f0); o.x += y[j].x * whole(f0); o.z += y[j].z * whole(f0);
        l1 += w[j].w * f1 * rest(f1); o.y += y[j].y * whole(f1); o.w += y[j].w * whole(f1);
      }
    }
    if (split > 1) {
      __syncthreads();                         // (the round before has been read)
      sum_o[warp][lane] = o;
      if (g == 0) sum_ml[warp][t] = make_float4(m0, l0, m1, l1);
      __syncthreads();
      if (warp % split != 0) continue;
      float n0 = m0, n1 = m1;
      for (int v = 1; v < split; ++v) { n0 = fmaxf(n0, sum_ml[warp + v][t].x); n1 = fmaxf(n1, sum_ml[warp + v][t].z); }
      o = make_float4(0.f, 0.f, 0.f, 0.f);
      l0 = l1 = 0.f;
      for (int v = 0; v < split; ++v) {
        const float4 y = sum_o[warp + v][lane], z = sum_ml[warp + v][t];
        const float f0 = factor(z.x, n0), f1 = factor(z.z, n1);
        l0 += z.y * f0 * rest(f0); o.x += y.x * whole(f0); o.z += y.z * whole(f0);
        l1 += z.w * f1 * rest(f1); o.y += y.y * whole(f1); o.w += y.w * whole(f1);
      }
    }
    if (k >= mine) continue;
    const int d = paged_dim<D, FP8>(g, q % MD), kh = p.groups == 1 ? item : item / p.groups, col0 = (item - kh * p.groups) * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = col0 + 2 * pair + h;
      const float l = h ? l1 : l0, inv = l == 0.f ? 0.f : (FP8 ? 1 << PAGED_SUM : 1) / l;
      if (c < s.rows * p.G)
        *reinterpret_cast<uint32_t*>(p.o + (s.row0 + c / p.G) * p.o_ld + (kh * p.G + c % p.G) * p.o_head + d) =
            h ? pack_bf16(o.y * inv, o.w * inv) : pack_bf16(o.x * inv, o.z * inv);
    }
  }
}

template <int D, bool FP8, int NT>
static int launch_paged_decode(PagedAttnParams& p, cudaStream_t st) {
  constexpr int smem = paged_decode_smem<D, NT>();
  static bool attr_set[64] = {false};
  int dev = 0;
  SB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    SB_CHECK_CUDA(cudaFuncSetAttribute(paged_decode_kernel<D, FP8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set[dev & 63] = true;
  }
  // Programmatic dependent launches: the first grid does nothing before `griddepcontrol.wait`, the second reads the batch's
  // description before it, which was complete before the first one ran.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(PD_WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, FP8, NT>, static_cast<const PagedAttnParams>(p)));
  if (p.part != nullptr) {
    cfg.gridDim = dim3(p.ctas - 1);
    cfg.blockDim = dim3(PJ_WARPS * 32);
    cfg.dynamicSmemBytes = 0;
    SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<D, FP8, NT>, static_cast<const PagedAttnParams>(p)));
  }
  return SB_OK;
}

// CTAs of a call: as many as fit the GPU at a time (two to an SM), and no more than there can be places of work. *cut: whether a
// (sequence, kv head) may be cut.
static int paged_decode_ctas(int B, int items, long keys, int D, bool fp8, bool* cut) {
  const int unit = PD_WARPS * (PD_STAGE / 2 / (fp8 ? D : 2 * D));
  const long units = (keys + unit - 1) / unit;
  const long ctas = min(static_cast<long>(B) * items * (units <= PD_WHOLE ? 1 : units), 2L * num_sms());
  *cut = units > PD_WHOLE && ctas > 1;
  return static_cast<int>(ctas);
}

}  // namespace sb

// fp32 elements of workspace that sb_paged_attention needs for `columns` = max_rows * Hq / Hkv; 0: none, `work` may be null.
extern "C" long sb_paged_attention_workspace(int B, int Hkv, int P, int page, int D, int fp8, int columns) {
  bool cut;
  const int ctas = sb::paged_decode_ctas(B, Hkv * ((columns + 15) / 16), static_cast<long>(P) * page, D, fp8 != 0, &cut);
  return cut ? 2L * ctas * (columns <= 8 ? 8 : 16) * (D + 2) : 0;
}

// The rows of the call are in the cache already: row i of sequence b stands at lengths[b] + i and sees the keys j < lengths[b] + rows,
// with causal those j <= its own position, with window >= 0 those |j - position| <= window. max_rows * Hq / Hkv is at most 48.
extern "C" int sb_paged_attention(const sb::PagedAttentionArgs* args) {
  using namespace sb;
  SB_CHECK_ARG(args != nullptr);
  const PagedAttentionArgs& c = *args;
  const int shift = page_shift_of(c.page);
  SB_CHECK_ARG((c.D == 64 || c.D == 128) && shift >= 0 && c.Hq > 0 && c.Hkv > 0 && c.Hq % c.Hkv == 0 && c.T > 0 && c.B > 0 && c.P > 0 && c.num_pages > 0);
  SB_CHECK_ARG(c.max_rows > 0 && (c.starts != nullptr || (c.T == c.B && c.max_rows == 1)) && (c.k_scale == nullptr) == (c.v_scale == nullptr));
  SB_CHECK_ARG(aligned16(c.q, c.k, c.v, c.o, c.work) && (c.q_ld | c.q_head | c.o_ld | c.o_head) % 8 == 0);
  SB_CHECK_ARG(c.max_rows <= 48 && c.max_rows * (c.Hq / c.Hkv) <= 48);
  const int groups = (c.max_rows * (c.Hq / c.Hkv) + 15) / 16;
  // places of the list of work in 32 bits, at the shortest unit; a page's stride in 32 bits (unsigned)
  SB_CHECK_ARG((static_cast<double>(c.P) * c.page / 64 + 1 + PD_START) * c.B * c.Hkv * groups < 2e9);
  const bool fp8 = c.k_scale != nullptr;
  const long size = fp8 ? 1 : 2;
  SB_CHECK_ARG(c.k_page >= 0 && c.v_page >= 0 && c.k_head >= 0 && c.v_head >= 0 && c.k_page * size < (1L << 32) && c.v_page * size < (1L << 32));
  PagedAttnParams p;
  p.batch = PagedBatch{c.table, c.lengths, c.starts, c.table_ld, c.P, c.B, c.T, c.max_rows, shift, c.num_pages};
  p.q = static_cast<const __nv_bfloat16*>(c.q); p.q_ld = c.q_ld; p.q_head = c.q_head;
  p.o = static_cast<__nv_bfloat16*>(c.o); p.o_ld = c.o_ld; p.o_head = c.o_head;
  p.k = static_cast<const uint8_t*>(c.k); p.v = static_cast<const uint8_t*>(c.v);
  p.k_page = c.k_page * size; p.k_head = c.k_head * size; p.v_page = c.v_page * size; p.v_head = c.v_head * size;
  p.ks = c.k_scale; p.vs = c.v_scale; p.ks_ld = c.k_scale_ld; p.vs_ld = c.v_scale_ld;
  p.Hq = c.Hq; p.Hkv = c.Hkv; p.G = c.Hq / c.Hkv; p.groups = groups;
  p.causal = c.causal; p.window = c.window; p.scale_log2 = c.scale * 1.4426950408889634f;
  p.zero_tail = c.zero_tail;
  bool cut;
  p.ctas = paged_decode_ctas(c.B, c.Hkv * groups, static_cast<long>(c.P) * c.page, c.D, fp8, &cut);
  SB_CHECK_ARG(!cut || c.work != nullptr);
  p.part = cut ? c.work : nullptr;
  p.err = error_word();
  if (!p.err) return SB_ERR_CUDA;
  const bool two = c.max_rows * p.G > 8;
#define SB_PD(DD, FF) return two ? launch_paged_decode<DD, FF, 2>(p, c.stream) : launch_paged_decode<DD, FF, 1>(p, c.stream)
  if (c.D == 64) { if (fp8) SB_PD(64, true); else SB_PD(64, false); }
  if (fp8) SB_PD(128, true);
  SB_PD(128, false);
#undef SB_PD
}
