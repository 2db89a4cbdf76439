// Attention of many query rows per sequence over the paged cache: prompt chunks behind what the cache already holds, whole prompts of
// several sequences at once (bf16 or e4m3 pages, head_dim 64 or 128).
//
// The products are dense enough for the tensor cores to bound them, so they run on tcgen05 with the scores, the weights and the output
// in tensor memory. A tile is 256 (row, head) pairs of one sequence and one kv head, rows first: pair x is row x / G, query head x % G.
// All heads that share the kv head ride in one tile, so the keys and values that it takes from the cache, and expands, serve G times
// the rows, and a short chunk fills the tile. Two groups of 128 pairs take turns on the tensor core:
//   warps 0-3 / 4-7   first the query rows to shared memory; then a thread per pair: per block of 64 keys its scores from tensor memory,
//                     masks, running maximum, weights back into tensor memory as operand A of the next product; at the end its output
//                     row, through shared memory
//   warp 8            issues S = Q K^T
//   warp 9            issues O += P V
//   warp 10           brings the scales of a block's pages, and says whether they lie far apart (that said by the softmax threads, and the scales
//                     brought by a copying warp: 107, and 113 from memory, were 106 and 117)
//   warps 12-15       bring keys and values from their pages into the swizzled tiles that the products read: bf16 as 16-byte
//                     asynchronous copies, e4m3 through registers, where it becomes f16
// Tensor memory holds the two groups' O (256 columns), one buffer of 64 scores and two of packed weights each. The scores' buffer is free
// again as soon as the threads have them in registers, so the scores of the next block are computed while the threads are at this one,
// and the product with its weights while they are at the next; they wait for one only where their maximum makes them rescale O. (One
// buffer of 128 scores with the weights in place: 6500 cycles for 128 keys, 2300 of them each group's wait for its two products. Two
// buffers of 64, in place: 4200.) What bounds it: the four products of 64 keys and 256 pairs are 1540 cycles of the tensor cores, a block takes
// 2100 with bf16 pages and 2900 with e4m3 ones. The threads between the two products do (512 cycles of exponentials for each group, on the
// same units), and with e4m3 the warps that expand the codes. Both groups on 16 warps of half a row each were slower (125 to 180 us where
// this took 102 to 118), and so was fetching two blocks of codes ahead in registers (117 us for 105).
//
// Measured at 32 query heads over 8 kv heads of 128: a chunk of 512 rows behind 7500 tokens 107 us in e4m3 and 88 in bf16 pages (606 and
// 740 TFLOP/s) that lie in the L2 cache, 113 and 89 from memory: e4m3 codes are asked for one block ahead, in registers, bf16 ones two by
// asynchronous copies. 256 rows behind 16000 tokens with 37 kv heads, a tile for every SM, 450 and 400 us (694 and 780); six prompts of
// 200 to 2048 rows in bf16 105 us, 16 rows behind 4000 tokens in e4m3 20.7.
//
// (A bulk tensor copy could fetch bf16 pages, but not expand codes, nor leave out single rows of a page that hold nothing yet: what
// lies behind a sequence's last row may be NaN, and 0 * NaN would reach its sums.)
//
// 8 bits: as in paged_attention.cu, codes enter the products as f16, a query row scaled by a power of two to at most 2^15, the key
// scale of each 16 keys in the factor of the scores, the value scale 2^e in the weight w = 2^(s + e - M), beside the sum of 2^(s - M),
// which is that of w 2^-e, or comes from the scores where pages lie far apart. With bf16 pages the factor is the softmax scale, e is
// 0, and the weights are rounded to bf16, since both operands of a product have one type and the values are bf16.
// Keys that a sequence has no page for have a score of -infinity.
//
// With few tiles the keys are split too: each of `splits` CTAs takes a part of the tile's blocks and leaves O (unnormalised, 32
// bits), M and l; a second kernel adds them up in order. (Dealing out equal stretches of all tiles' blocks to one CTA per SM instead, the
// next tile's queries fetched during the last block of one, took 111 us for the 105 of the chunk and 152 for the 127 of the prompts in
// e4m3: a change of tile costs such a CTA as much as a new one, 10,000 cycles, and the cuts come on top. Two groups that share the
// keys of a tile of 128 pairs gained nothing below 128 pairs: there the copying warps are the bound.)
#include "paged.cuh"

namespace sb {

struct PagedPrefillParams {
  PagedBatch batch;
  const __nv_bfloat16* q;
  long q_ld, q_head;
  __nv_bfloat16* o;
  long o_ld, o_head;
  const uint8_t *k, *v;
  long k_page, k_head, v_page, v_head;     // bytes
  const float *ks, *vs;
  long ks_ld, vs_ld;
  int Hq, Hkv, G;
  int causal, window;
  float scale_log2;
  int zero_tail, splits, tiles;            // tiles: the most that the rows of the call can need
  float* part;                             // [splits][tiles][Hkv]: [256][D] of O, then [256][2] of (m, l)
  unsigned int* err;
};

constexpr int PP_THREADS = 512, PP_KEYS = 64;
constexpr int PP_JOIN = 16;     // blocks of the second kernel for a tile, a pair or two per warp: 105 us for the chunk, 112 with 4

template <int D, bool FP8>
struct PagedPrefill {
  static constexpr int TILE = 128 * D * 2, KTILE = PP_KEYS * D * 2;
  static constexpr int NS = 4;                                   // stages of keys and of values
  static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + NS * KTILE, OFF_SCALE = OFF_V + NS * KTILE;
  static constexpr int RING = 8;                                 // blocks whose scales are kept: more than can be under way
  static constexpr int OFF_BACK = OFF_SCALE + RING * 4 * 16;     // [256] floats: the rows' factors
  static constexpr int OFF_BAR = OFF_BACK + 1024;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static constexpr int COL_P = 128, COL_O = 256;                 // S of group a at a * 64, P at COL_P + (a * 2 + buffer) * 32, O at COL_O + a * D
  static constexpr int CPR = (FP8 ? D : 2 * D) / 16;             // 16-byte chunks of a key
  static constexpr int LOADS = PP_KEYS * CPR / 128;              // of a copying thread, per tile of 64 keys
  static constexpr float HEAD = FP8 ? 9.f : 0.f, SLACK = FP8 ? 6.f : 8.f;
};

// f16 operands: as make_idesc_bf16, formats 0
__host__ __device__ constexpr uint32_t make_idesc_f16(int M, int N, int a_mn_major, int b_mn_major) {
  return make_idesc_bf16(M, N, a_mn_major, b_mn_major) & ~((1u << 7) | (1u << 10));
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

struct PrefillTile {
  int b, tile;                      // of sequence b
  int row0, rows, len, hi;          // its rows of the call, tokens before, keys in the cache
};

// The tile-th tile of the call (b = B behind the last). By a whole warp.
__device__ __forceinline__ PrefillTile prefill_tile(const PagedBatch& p, int G, int tile) {
  const int lane = threadIdx.x & 31;
  PrefillTile r;
  r.b = p.B; r.tile = 0; r.row0 = r.rows = r.hi = 0; r.len = -1;
  int front = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int rows = b0 + lane < p.B ? paged_seq(p, b0 + lane).rows : 0;
    const int n = (static_cast<unsigned>(rows) * G + 255) / 256;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned in_front = __ballot_sync(0xffffffffu, front + sum <= tile);
    if (in_front != 0xffffffffu) {
      const int l = __popc(in_front);
      r.b = b0 + l;
      // tiles of a sequence from the last to the first: with a causal mask the last has the most keys, and starts first
      const int at = tile - front - __shfl_sync(0xffffffffu, sum - n, l);
      r.tile = __shfl_sync(0xffffffffu, n, l) - 1 - at;
      break;
    }
    front += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (r.b < p.B) {
    const PagedSeq s = paged_seq(p, r.b);
    r.row0 = s.row0; r.rows = s.rows; r.len = s.len;
    const long cap = min(static_cast<long>(p.P) << p.page_shift, 0x7fffff00L);
    r.hi = s.len < 0 ? 0 : static_cast<int>(min(static_cast<long>(s.len) + s.rows, cap));
  }
  return r;
}

template <int D, bool FP8>
__global__ void __launch_bounds__(PP_THREADS, 1) paged_prefill_kernel(const PagedPrefillParams p) {
  using C = PagedPrefill<D, FP8>;
  constexpr int NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  // (where threads arrive, a warp's have fenced what they did, and one of them does)
  uint64_t* q_full = bars + 0;    // 8 arrivals
  uint64_t* s_full = bars + 1;    // [2]
  uint64_t* s_free = bars + 3;    // [2], 4 arrivals: the group has its scores in registers
  uint64_t* p_full = bars + 5;    // [2][2 buffers], 4 arrivals
  uint64_t* o_full = bars + 9;    // [2][2] the product with a buffer's weights is complete (one for each buffer: who waits is a phase behind at most)
  uint64_t* k_full = bars + 13;   // [NS], 5 arrivals: the keys', and their scales'
  uint64_t* k_empty = bars + 17;
  uint64_t* v_full = bars + 21;   // [NS], 4 arrivals
  uint64_t* v_empty = bars + 25;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 29);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float4* scales = reinterpret_cast<float4*>(smem + C::OFF_SCALE);       // [RING][4]: key factor, e, 2^(PAGED_SUM - e), whether the block's pages are far apart

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kh = blockIdx.x;
  const PrefillTile tl = prefill_tile(p.batch, p.G, blockIdx.y);
  // rows behind the last sequence: thread i0 of as many in every CTA, with a tile or without (so that together they take all of them)
  constexpr int n0 = 128;
  auto zero_tail = [&](int i0) {
    if (!p.zero_tail) return;
    const int t0 = paged_tail(p.batch);
    const long n = static_cast<long>(p.batch.T - t0) * p.Hq * (D / 8);
    const long cta = blockIdx.x + static_cast<long>(gridDim.x) * (blockIdx.y + static_cast<long>(gridDim.y) * blockIdx.z);
    const long ctas = static_cast<long>(gridDim.x) * gridDim.y * gridDim.z;
    for (long i = cta * n0 + i0; i < n; i += ctas * n0) {
      const long row = i / (p.Hq * (D / 8));
      const int x = static_cast<int>(i % (p.Hq * (D / 8)));
      *reinterpret_cast<uint4*>(p.o + (t0 + row) * p.o_ld + (x / (D / 8)) * p.o_head + (x % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
  };
  if (tl.b >= p.batch.B) {
    if (threadIdx.x < n0) zero_tail(threadIdx.x);
    return;
  }

  // the tile's pairs and the keys that any of them sees
  const unsigned pairs = static_cast<unsigned>(tl.rows) * p.G, x0 = static_cast<unsigned>(tl.tile) * 256, G = p.G;
  const int tiles_here = pairs - x0 > 128 ? 2 : 1;               // groups that have pairs
  const int first_row = x0 / G, last_row = (min(pairs, x0 + 256) - 1) / G;
  int lo = 0, hi = tl.hi;
  if (tl.len >= 0) {
    if (p.causal) hi = static_cast<int>(min(static_cast<long>(hi), static_cast<long>(tl.len) + last_row + 1));
    else if (p.window >= 0) hi = static_cast<int>(min(static_cast<long>(hi), static_cast<long>(tl.len) + last_row + p.window + 1));
    // (a length may be anything: behind the last key there is none, whatever 32 bits hold)
    if (p.window >= 0) lo = static_cast<int>(min(max(static_cast<long>(tl.len) + first_row - p.window, 0L), static_cast<long>(hi)));
  }
  int j0 = lo / PP_KEYS, j1 = (hi + PP_KEYS - 1) / PP_KEYS;       // blocks of keys
  if (hi <= lo) j1 = j0;
  if (p.splits > 1) {
    const int per = (j1 - j0 + p.splits - 1) / p.splits, end = j1;
    j0 = min(j0 + static_cast<int>(blockIdx.z) * per, end);
    j1 = min(j0 + per, end);
  }
  const int nblk = j1 - j0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < 4; ++s) { mbar_init(&p_full[s], 4); mbar_init(&o_full[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&s_full[a], 1); mbar_init(&s_free[a], 4); }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 5); mbar_init(&k_empty[s], 1); mbar_init(&v_full[s], 4); mbar_init(&v_empty[s], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    if (tl.hi < static_cast<long>(tl.len) + tl.rows && tl.len >= 0) atomicOr(p.err, 4u);      // positions behind the table's end
  }
  if (warp == 9) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 12) {
    // ---------------------------------------------------------------- copies
    // Chunk x of a thread is row x * RPI + r0 of the tile, chunk c of the row; 16 rows of one page share a look-up, done a block ahead.
    const int tid = threadIdx.x - 384, shift = p.batch.page_shift, mask = (1 << shift) - 1;
    const int* table = p.batch.table + tl.b * p.batch.table_ld;
    constexpr int ROWB = C::CPR * 16, RPI = 128 / C::CPR, LOADS = C::LOADS, IDS = RPI >= 16 ? LOADS : 4;
    const int r0 = tid / C::CPR, c = tid % C::CPR, group0 = RPI >= 16 ? r0 & ~15 : 0;      // first row of id 0's group
    constexpr int IDROWS = RPI >= 16 ? RPI : 16;                                           // rows between two ids' groups
    const uint32_t lane_off = (r0 - group0) * ROWB + c * 16;
    const uint8_t *kb = p.k + kh * p.k_head + lane_off, *vb = p.v + kh * p.v_head + lane_off;
    const unsigned pages = p.batch.num_pages;
    int id[IDS], next[IDS];
    auto look_up = [&](int j) {
#pragma unroll
      for (int i = 0; i < IDS; ++i) {
        const int key = j * PP_KEYS + i * IDROWS + group0;
        next[i] = -2;
        if (j < j1 && key + 16 > lo && key < hi) next[i] = table[key >> shift];
      }
    };
    // Copies of block j through take(x, source, whether it is a key of the sequence). Where all of them are, the addresses of a group are
    // one multiplication and constants.
    auto each = [&](const uint8_t* base, long stride, int j, auto take) {
      bool all = j * PP_KEYS >= lo && (j + 1) * PP_KEYS <= hi;
#pragma unroll
      for (int i = 0; i < IDS; ++i) all = all && static_cast<unsigned>(id[i]) < pages;
      if (all) {
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
          const uint8_t* src = base + (static_cast<uint64_t>(static_cast<uint32_t>(id[i])) * static_cast<uint32_t>(stride) +
                                       static_cast<uint32_t>(((j * PP_KEYS + i * IDROWS + group0) & mask) * ROWB));
#pragma unroll
          for (int x = 0; x < LOADS / IDS; ++x) take(i * (LOADS / IDS) + x, src + x * RPI * ROWB, true);
        }
      } else {
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
          const int key = j * PP_KEYS + i * IDROWS + group0;
          const bool good = static_cast<unsigned>(id[i]) < pages;
          const uint8_t* src = base + (good ? static_cast<uint64_t>(static_cast<uint32_t>(id[i])) * static_cast<uint32_t>(stride) +
                                              static_cast<uint32_t>((key & mask) * ROWB) : 0);
#pragma unroll
          for (int x = 0; x < LOADS / IDS; ++x) {
            const int at = key + (r0 - group0) + x * RPI;
            const bool in = good && at >= lo && at < hi;
            take(i * (LOADS / IDS) + x, in ? src + x * RPI * ROWB : p.k, in);
          }
        }
      }
    };
    // where elements 8 e .. 8 e + 7 of row r lie in a tile: 64 elements a row of a swizzled half
    auto place = [&](int r, int e) -> uint32_t { return (e >> 3) * (PP_KEYS * 128) + r * 128 + (((e & 7) ^ (r & 7)) << 4); };
    auto turn = [&](int j) {                     // to block j
#pragma unroll
      for (int x = 0; x < IDS; ++x) id[x] = next[x];
      look_up(j + 1);
    };
    bool ok = true;
    look_up(j0);
    if (FP8) {
      uint4 rk[LOADS], rv[LOADS];
      auto load = [&](uint4* r, const uint8_t* base, long stride, int j) {
        each(base, stride, j, [&](int x, const uint8_t* src, bool in) {
          if (in) r[x] = *reinterpret_cast<const uint4*>(src);
          else r[x] = make_uint4(0, 0, 0, 0);
        });
      };
      auto store = [&](const uint4* r, uint8_t* dst) {
#pragma unroll
        for (int x = 0; x < LOADS; ++x) {
          const uint32_t w[4] = {r[x].x, r[x].y, r[x].z, r[x].w};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
                : "=r"(h[2 * k]), "=r"(h[2 * k + 1]) : "r"(w[k]));
          // (where a row goes to two swizzled halves, the upper half's threads begin with the second 8 elements: the halves share banks)
          const bool upper = 2 * c >= 8;
          *reinterpret_cast<uint4*>(dst + place(x * RPI + r0, 2 * c + (upper ? 1 : 0))) =
              upper ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(dst + place(x * RPI + r0, 2 * c + (upper ? 0 : 1))) =
              upper ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]);
        }
        fence_proxy_async_smem();
      };
      turn(j0);
      if (nblk > 0) load(rk, kb, p.k_page, j0);
      for (int i = 0; i < nblk && ok; ++i) {
        const int s = i % NS;
        load(rv, vb, p.v_page, j0 + i);
        ok = mbar_wait(&k_empty[s], ((i / NS) & 1) ^ 1, abort_flag, p.err);
        if (!ok) break;
        store(rk, smem + C::OFF_K + s * C::KTILE);
        warp_arrive(&k_full[s]);
        turn(j0 + i + 1);
        if (i + 1 < nblk) load(rk, kb, p.k_page, j0 + i + 1);
        ok = mbar_wait(&v_empty[s], ((i / NS) & 1) ^ 1, abort_flag, p.err);
        if (!ok) break;
        store(rv, smem + C::OFF_V + s * C::KTILE);
        warp_arrive(&v_full[s]);
      }
    } else {
      // tiles in the order K of block 0, V of block 0, K of block 1, ...; one is handed over when the two behind it are under way
      auto full = [&](int n) { return (n & 1) ? &v_full[(n >> 1) % NS] : &k_full[(n >> 1) % NS]; };
      for (int n = 0; n < 2 * nblk && ok; ++n) {
        const int i = n >> 1, j = j0 + i, s = i % NS;
        const bool is_v = n & 1;
        if (!is_v) turn(j);
        ok = mbar_wait(is_v ? &v_empty[s] : &k_empty[s], ((i / NS) & 1) ^ 1, abort_flag, p.err);
        if (!ok) break;
        uint8_t* dst = smem + (is_v ? C::OFF_V : C::OFF_K) + s * C::KTILE;
        const uint32_t at = smem_u32(dst) + place(r0, c);
        each(is_v ? vb : kb, is_v ? p.v_page : p.k_page, j, [&](int x, const uint8_t* src, bool in) {
          // (rows x * RPI: the swizzle of r0's)
          cp_async16_zfill(at + x * RPI * 128, src, in ? 16 : 0);
        });
        cp_async_commit();
        if (n >= 2) {
          cp_async_wait_group<2>();
          fence_proxy_async_smem();
          warp_arrive(full(n - 2));
        }
      }
      cp_async_wait_group<0>();
      if (ok && nblk > 0) {
        fence_proxy_async_smem();
        warp_arrive(full(2 * nblk - 2));
        warp_arrive(full(2 * nblk - 1));
      }
    }
    zero_tail(tid);
  } else if (warp >= 8) {
    // (whole warps go through these loops and one elected thread issues, so that the descriptors, the same for all, stay in uniform
    // registers: from a lane of its own an instruction took 100 cycles to issue)
    if (warp == 8 && nblk > 0) {
      // -------------------------------------------------------------- S = Q K^T
      constexpr uint32_t idesc = FP8 ? make_idesc_f16(128, PP_KEYS, 0, 0) : make_idesc_bf16(128, PP_KEYS, 0, 0);
      const uint64_t q_desc = make_smem_desc_sw128(smem_u32(smem), 16, 1024), k_desc = make_smem_desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
      bool ok = mbar_wait(q_full, 0, abort_flag, p.err);
      for (int i = 0; i < nblk && ok; ++i) {
        const int ks = i % NS;
        ok = mbar_wait(&k_full[ks], (i / NS) & 1, abort_flag, p.err);
        for (int a = 0; a < tiles_here && ok; ++a) {
          if (i > 0) ok = mbar_wait(&s_free[a], (i - 1) & 1, abort_flag, p.err);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_fence_after();
          const uint64_t qa = q_desc + a * (C::TILE >> 4), kb = k_desc + ks * (C::KTILE >> 4);       // (addresses in 16 bytes)
          const uint32_t to = tmem_base + a * 64;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_bf16(to, qa + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), kb + (((kk >> 2) * (PP_KEYS * 128) + (kk & 3) * 32) >> 4), idesc,
                        kk > 0 ? 1u : 0u);
            umma_commit(&s_full[a]);
            if (a == tiles_here - 1) umma_commit(&k_empty[ks]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 9 && nblk > 0) {
      // -------------------------------------------------------------- O += P V
      constexpr uint32_t idesc = FP8 ? make_idesc_f16(128, D, 0, 1) : make_idesc_bf16(128, D, 0, 1);
      const uint64_t v_desc = make_smem_desc_sw128(smem_u32(smem + C::OFF_V), PP_KEYS * 128, 1024);
      bool ok = true;
      for (int i = 0; i < nblk && ok; ++i) {
        const int vs = i % NS, b = i & 1;
        ok = mbar_wait(&v_full[vs], (i / NS) & 1, abort_flag, p.err);
        for (int a = 0; a < tiles_here && ok; ++a) {
          ok = mbar_wait(&p_full[a * 2 + b], (i >> 1) & 1, abort_flag, p.err);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_fence_after();
          const uint64_t vd = v_desc + vs * (C::KTILE >> 4);
          const uint32_t to = tmem_base + C::COL_O + a * D, from = tmem_base + C::COL_P + (a * 2 + b) * 32;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < PP_KEYS / 16; ++kk)
              umma_bf16_ta(to, from + 8 * kk, vd + ((kk * 2048) >> 4), idesc, (i > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&o_full[a * 2 + b]);
            if (a == tiles_here - 1) umma_commit(&v_empty[vs]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 10 && nblk > 0) {
      // -------------------------------------------------------------- scales
      // Of a block's groups of 16 keys, read by the softmax threads behind S: a lane for each group. Short of 2^100 between the scales of a
      // block's pages and those in front of them a share of the sum l down to 2^-25 of the largest has a weight of 2^(e - the largest e - 16) or
      // more, which 32 bits hold; a block with a page further below the largest so far is marked.
      const int* table = p.batch.table + tl.b * p.batch.table_ld;
      const unsigned pages = p.batch.num_pages;
      auto look_up = [&](int j) {                // -2: no key of the sequence; others out of range: no page
        const int key = j * PP_KEYS + lane * 16;
        return lane < 4 && j < j1 && key + 16 > lo && key < hi ? table[key >> p.batch.page_shift] : -2;
      };
      int id = look_up(j0), top_e = PAGED_LEAST_EXP;
      bool ok = true;
      for (int i = 0; i < nblk && ok; ++i) {
        const int page = id;
        const bool good = static_cast<unsigned>(page) < pages;
        id = look_up(j0 + i + 1);
        if (!good && page != -2) atomicOr(p.err, 4u);
        float4 f = make_float4(1.f, 0.f, good ? 1.f : 0.f, 0.f);
        if (FP8) {
          float vs = 1.f;
          if (good) { f.x = p.ks[page * p.ks_ld + kh]; vs = p.vs[page * p.vs_ld + kh]; }
          const int e = min(max(scale_exp(vs), PAGED_LEAST_EXP), PAGED_MOST_EXP);
          const int least = __reduce_min_sync(0xffffffffu, good ? e : PAGED_MOST_EXP);
          top_e = max(top_e, __reduce_max_sync(0xffffffffu, good ? e : PAGED_LEAST_EXP));
          if (good) { f.y = static_cast<float>(e); f.z = exp_scale(PAGED_SUM - e); }
          f.w = least + 100 < top_e ? 1.f : 0.f;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[i % NS], ((i / NS) & 1) ^ 1, abort_flag, p.err));
        if (!ok) break;
        if (lane < 4) scales[(i % C::RING) * 4 + lane] = f;
        warp_arrive(&k_full[i % NS]);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax, a thread per pair
    const int a = warp >> 2, t = threadIdx.x & 127;
    const unsigned x = x0 + a * 128 + t;
    const bool live = x < pairs;
    const int row = live ? x / G : 0;
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem_base + a * 64 + lane_sel, t_o = tmem_base + C::COL_O + a * D + lane_sel;

    // The query rows into the group's tile, a warp its own 32: D / 8 threads a row. In 8 bits a thread then turns its row to f16, scaled by a
    // power of two, whose inverse it keeps. (What runs once per tile is kept in short loops: unrolled over registers this was 11,000 cycles of
    // a tile, most of them instruction fetches.)
    const uint32_t back_at = smem_u32(smem + C::OFF_BACK) + threadIdx.x * 4;
    const int wr = warp & 3;
    // (the tile's first row stands in for a pair that is none)
    auto pair_offset = [&](long ld, long head_ld) { return (tl.row0 + (live ? x : x0) / G) * ld + (kh * G + (live ? x : x0) % G) * head_ld; };
    if (a < tiles_here) {
      constexpr int TPR = D / 8, RPS = 32 / TPR;
      const int c = lane % TPR;
      const long mine = pair_offset(p.q_ld, p.q_head);
      const unsigned there = __ballot_sync(0xffffffffu, live);
      uint8_t* tile = smem + a * C::TILE + wr * 32 * 128;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += RPS) {
        const int r = r0 + lane / TPR;
        const long at = __shfl_sync(0xffffffffu, mine, r);
        cp_async16_zfill(smem_u32(tile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)), p.q + at + c * 8, there >> r & 1 ? 16 : 0);
      }
      cp_async_commit();
      cp_async_wait_group<0>();
      if (FP8) {
        __syncwarp();
        __nv_bfloat162 most2 = __float2bfloat162_rn(0.f);
        auto chunk = [&](int k) { return reinterpret_cast<uint4*>(tile + (k >> 3) * 16384 + lane * 128 + (((k & 7) ^ (lane & 7)) << 4)); };
#pragma unroll 4
        for (int k = 0; k < TPR; ++k) {
          const uint4 w = *chunk(k);
          const uint32_t u[4] = {w.x & 0x7fff7fffu, w.y & 0x7fff7fffu, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu};
#pragma unroll
          for (int i = 0; i < 4; ++i) most2 = __hmax2(most2, *reinterpret_cast<const __nv_bfloat162*>(&u[i]));
        }
        const float most = fmaxf(__low2float(most2), __high2float(most2));
        int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100);
        if (most == 0.f || !(most < INFINITY)) e = 14;
        const float mul = exp_scale(14 - e);
        asm volatile("st.shared.f32 [%0], %1;" :: "r"(back_at), "f"(p.scale_log2 * exp_scale(e - 14)) : "memory");
#pragma unroll 2
        for (int k = 0; k < TPR; ++k) {
          const uint4 w = *chunk(k);
          uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(bf16_lo(u[i]) * mul, bf16_hi(u[i]) * mul);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *chunk(k) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
      fence_proxy_async_smem();
    }
    warp_arrive(q_full);

    // keys that this pair sees: [klo, khi)
    const long pos = static_cast<long>(tl.len) + row;
    int klo = 0, khi = tl.hi;
    if (p.causal) khi = static_cast<int>(min(static_cast<long>(khi), pos + 1));
    if (p.window >= 0) {
      klo = static_cast<int>(min(max(pos - p.window, 0L), static_cast<long>(khi)));
      khi = static_cast<int>(min(static_cast<long>(khi), pos + p.window + 1));
    }
    if (!live) khi = 0;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = a < tiles_here;
#pragma unroll 1
    for (int i = 0; i < nblk && ok; ++i) {
      const int kv0 = (j0 + i) * PP_KEYS, b = i & 1;
      if (!mbar_wait(&s_full[a], i & 1, abort_flag, p.err)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[64];
      tmem_ld_32x32b_x32(t_s, v);
      tmem_ld_32x32b_x32(t_s + 32, v + 32);
      // factor and exponent of the four groups of 16 keys (bf16 pages: the softmax scale and 0)
      const uint32_t sc = smem_u32(scales) + (i % C::RING) * 64;
      float fs[4], e[4], inv[4];
      float back = p.scale_log2;
      if (FP8) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(back) : "r"(back_at) : "memory");
      bool masked = kv0 < klo || kv0 + PP_KEYS > khi;
#pragma unroll
      for (int gp = 0; gp < 4; ++gp) {
        float unused;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(fs[gp]), "=f"(e[gp]), "=f"(inv[gp]), "=f"(unused) : "r"(sc + gp * 16) : "memory");
        masked |= inv[gp] == 0.f;              // a page is missing
        fs[gp] = FP8 ? fs[gp] * back : back;
      }
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(&s_free[a]);
      if (masked) {
        const int from = klo - kv0, to = khi - kv0;
#pragma unroll
        for (int k = 0; k < 64; ++k) v[k] = (k >= from && k < to && inv[k >> 4] != 0.f) ? v[k] : 0xff800000u;   // -inf
#pragma unroll
        for (int gp = 0; gp < 4; ++gp) fs[gp] = fmaxf(fs[gp], 1e-37f);     // (-inf times what has underflown to 0 would be NaN)
      }
      float m_blk = -INFINITY;
#pragma unroll
      for (int gp = 0; gp < 4; ++gp) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < 16; k += 2) mx = fmaxf(mx, fmaxf(__uint_as_float(v[gp * 16 + k]), __uint_as_float(v[gp * 16 + k + 1])));
        m_blk = fmaxf(m_blk, FP8 ? fmaf(mx, fs[gp], e[gp]) : mx * fs[gp]);
      }
      const bool grow = m_blk > m_ref + C::SLACK;
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = grow ? m_blk : m_ref;
        const float half = !grow ? 1.f : m_ref == -INFINITY ? 0.f : FP8 ? exp2_half(m_ref, m_new) : fast_exp2(m_ref - m_new);
        const float alpha = FP8 ? half * half : half;
        l *= half;
        if (FP8) l *= half;
        m_ref = m_new;
        if (i > 0) {
          // O is at rest once the product of the block before is complete: this block's waits for its weights
          if (!mbar_wait(&o_full[a * 2 + (b ^ 1)], ((i - 1) >> 1) & 1, abort_flag, p.err)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t o16[16];
            tmem_ld_32x32b_x16(t_o + cc * 16, o16);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o16[k] = __float_as_uint(__uint_as_float(o16[k]) * alpha);
            tmem_st_32x32b_x16(t_o + cc * 16, o16);
          }
        }
      }
      // this buffer's weights of two blocks ago have been used
      if (i > 1) {
        if (!mbar_wait(&o_full[a * 2 + b], ((i - 2) >> 1) & 1, abort_flag, p.err)) { ok = false; break; }
        tc_fence_after();
      }
      const float nm = C::HEAD - (m_ref == -INFINITY ? 0.f : m_ref);
      if (FP8) {
        // (of pages far apart in scale the one's w is nothing beside the other's, its share of l is not: then l comes from the scores)
        float apart;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(apart) : "r"(sc + 12) : "memory");
        if (__builtin_expect(apart != 0.f, 0)) {
#pragma unroll
          for (int k = 0; k < 64; ++k) l += inv[k >> 4] != 0.f ? fast_exp2(fmaf(__uint_as_float(v[k]), fs[k >> 4], nm + PAGED_SUM)) : 0.f;
          inv[0] = inv[1] = inv[2] = inv[3] = 0.f;
        }
      }
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t pk[16];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int gp = cc * 2 + hh;
          const float n1 = FP8 ? e[gp] + nm : nm;
          const uint64_t f2 = f2_pack(fs[gp], fs[gp]), n2 = f2_pack(n1, n1);
          uint64_t sum2 = f2_pack(0.f, 0.f);
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            const int k = gp * 16 + 2 * jj;
            float y0, y1;
            f2_unpack(f2_fma(f2_pack_u(v[k], v[k + 1]), f2, n2), y0, y1);
            const float e0 = fast_exp2(y0), e1 = fast_exp2(y1);
            sum2 = f2_add(sum2, f2_pack(e0, e1));
            if (FP8) {
              const __half2 h = __floats2half2_rn(e0, e1);
              pk[hh * 8 + jj] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              pk[hh * 8 + jj] = pack_bf16(e0, e1);
            }
          }
          float s0, s1;
          f2_unpack(sum2, s0, s1);
          l = FP8 ? fmaf(s0 + s1, inv[gp], l) : l + (s0 + s1);
        }
        tmem_st_32x32b_x16(tmem_base + C::COL_P + (a * 2 + b) * 32 + lane_sel + cc * 16, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&p_full[a * 2 + b]);
    }
    const bool have = ok && nblk > 0 && mbar_wait(&o_full[a * 2 + ((nblk - 1) & 1)], ((nblk - 1) >> 1) & 1, abort_flag, p.err);
    if (have) tc_fence_after();
    // The rows leave through shared memory (the group's query tile: its products are done), so that a row's bytes are stored side by
    // side; a warp has 32 rows of 2 D bytes there: a bf16 row, or half a row in 32 bits.
    constexpr int CH = D / 8;                    // 16-byte chunks of those
    uint8_t* stage = smem + a * C::TILE + wr * (32 * D * 2);
    const unsigned xw = x0 + a * 128 + (warp & 3) * 32;
    auto staged = [&](int r, int c) { return reinterpret_cast<uint4*>(stage + r * (D * 2) + ((c ^ (r & (CH - 1))) << 4)); };
    if (p.splits > 1) {
      const size_t at = ((static_cast<size_t>(blockIdx.z) * p.tiles + blockIdx.y) * p.Hkv + kh) * 256 + a * 128;
      float* ml = p.part + static_cast<size_t>(p.splits) * p.tiles * p.Hkv * 256 * D + (at + t) * 2;
      if (live) *reinterpret_cast<float2*>(ml) = make_float2(have ? m_ref : -INFINITY, have ? l : 0.f);
      if (__all_sync(0xffffffffu, have)) {       // (what has no keys is not read again)
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o16[16];
            tmem_ld_32x32b_x16(t_o + h * (D / 2) + cc * 16, o16);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 4; ++k) *staged(lane, cc * 4 + k) = make_uint4(o16[4 * k], o16[4 * k + 1], o16[4 * k + 2], o16[4 * k + 3]);
          }
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < CH; ++i) {
            const int r = i * (32 / CH) + lane / CH, c = lane % CH;
            if (xw + r < pairs)
              *reinterpret_cast<uint4*>(p.part + (at + (warp & 3) * 32 + r) * D + h * (D / 2) + c * 4) = *staged(r, c);
          }
          __syncwarp();
        }
      }
    } else {
      // At D = 128 a warp's rows of the stage are rows of another's queries. With keys those are at rest, since the last product is behind
      // them; a tile without a block of keys has no product, and its four warps meet here.
      if (nblk == 0) asm volatile("bar.sync %0, 128;" ::"r"(1 + a) : "memory");
      // (a sum of nothing: no key, zeros; a NaN stays one)
      const float inv_l = l == 0.f ? 0.f : (FP8 ? 1 << PAGED_SUM : 1) / l;
      const long mine = pair_offset(p.o_ld, p.o_head);
#pragma unroll 1
      for (int cc = 0; cc < D / 16; ++cc) {
        uint32_t o16[16];
        if (__all_sync(0xffffffffu, have)) {
          tmem_ld_32x32b_x16(t_o + cc * 16, o16);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o16[k] = 0u;
        }
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          uint4 w;
          w.x = pack_bf16(__uint_as_float(o16[k + 0]) * inv_l, __uint_as_float(o16[k + 1]) * inv_l);
          w.y = pack_bf16(__uint_as_float(o16[k + 2]) * inv_l, __uint_as_float(o16[k + 3]) * inv_l);
          w.z = pack_bf16(__uint_as_float(o16[k + 4]) * inv_l, __uint_as_float(o16[k + 5]) * inv_l);
          w.w = pack_bf16(__uint_as_float(o16[k + 6]) * inv_l, __uint_as_float(o16[k + 7]) * inv_l);
          *staged(lane, cc * 2 + k / 8) = w;
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int i = 0; i < CH; ++i) {
        const int r = i * (32 / CH) + lane / CH, c = lane % CH;
        const long at = __shfl_sync(0xffffffffu, mine, r);
        if (xw + r < pairs) *reinterpret_cast<uint4*>(p.o + at + c * 8) = *staged(r, c);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Adds up the parts of a tile: block (kv head, tile), a warp per pair, D / 32 dimensions a lane.
template <int D>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const PagedPrefillParams p) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kh = blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;");
  const PrefillTile tl = prefill_tile(p.batch, p.G, blockIdx.y);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tl.b >= p.batch.B) return;
  const unsigned pairs = static_cast<unsigned>(tl.rows) * p.G, x0 = static_cast<unsigned>(tl.tile) * 256, G = p.G;
  const size_t stride = static_cast<size_t>(p.tiles) * p.Hkv * 256;                 // pairs between two splits
  const float* ml0 = p.part + p.splits * stride * D;
  for (unsigned r = blockIdx.z * 8 + warp; r < 256 && x0 + r < pairs; r += 8 * gridDim.z) {
    const size_t at = (static_cast<size_t>(blockIdx.y) * p.Hkv + kh) * 256 + r;
    float top = -INFINITY, sum = 0.f, o[V] = {};
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, ml0[(s * stride + at) * 2]);
    for (int s = 0; s < p.splits; ++s) {
      const float2 w = *reinterpret_cast<const float2*>(ml0 + (s * stride + at) * 2);
      if (w.x == -INFINITY && w.y == 0.f) continue;      // no key there: its O was not written
      const float half = w.x == -INFINITY ? 0.f : exp2_half(w.x, top), f = half * half;
      sum += w.y * half * half;
      const float* y = p.part + (s * stride + at) * D + lane * V;
      if (V == 4) {
        const float4 z = *reinterpret_cast<const float4*>(y);
        o[0] += z.x * f; o[1] += z.y * f; o[2 % V] += z.z * f; o[3 % V] += z.w * f;
      } else {
        const float2 z = *reinterpret_cast<const float2*>(y);
        o[0] += z.x * f; o[1] += z.y * f;
      }
    }
    const float inv = sum == 0.f ? 0.f : (p.ks != nullptr ? 1 << PAGED_SUM : 1) / sum;
    __nv_bfloat16* dst = p.o + (tl.row0 + (x0 + r) / G) * p.o_ld + (kh * G + (x0 + r) % G) * p.o_head + lane * V;
    if (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2 % V] * inv, o[3 % V] * inv));
    else *reinterpret_cast<uint32_t*>(dst) = pack_bf16(o[0] * inv, o[1] * inv);
  }
}

template <int D, bool FP8>
static int launch_paged_prefill(PagedPrefillParams& p, cudaStream_t st) {
  using C = PagedPrefill<D, FP8>;
  static bool attr_set[64] = {false};
  int dev = 0;
  SB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    SB_CHECK_CUDA(cudaFuncSetAttribute(paged_prefill_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_set[dev & 63] = true;
  }
  // Programmatic dependent launches: the first grid does nothing before `griddepcontrol.wait`, the second reads the batch's
  // description before it, which was complete before the first one let it start.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.Hkv, p.tiles, p.splits);
  cfg.blockDim = dim3(PP_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_prefill_kernel<D, FP8>, static_cast<const PagedPrefillParams>(p)));
  if (p.splits > 1) {
    cfg.gridDim = dim3(p.Hkv, p.tiles, PP_JOIN);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<D>, static_cast<const PagedPrefillParams>(p)));
  }
  return SB_OK;
}

// Tiles that T rows of B sequences can need, and parts that the keys of a tile are split into: as many as make the rounds of CTAs over
// the GPU the shortest, a part costing two blocks of keys beside its own (a start, and its share of the join). A chunk of 512 rows behind 7500
// tokens (64 tiles): 178 us whole, 106 in two parts, which is what it comes to; 16 rows behind 4000 (8 tiles): 92 whole, 52 in two,
// 32 in four, 21 in sixteen.
static int paged_prefill_shape(int T, int B, int Hkv, int G, long keys, int* splits) {
  const long tiles = static_cast<long>(T) * G / 256 + min(B, T);
  const long items = tiles * Hkv, blocks = (keys + 127) / 128, sms = num_sms();
  long best = 0;
  *splits = 1;
  for (int s = 1; s <= 16 && s <= blocks; ++s) {
    const long cost = (items * s + sms - 1) / sms * ((blocks + s - 1) / s + (s > 1 ? 2 : 0));
    if (s == 1 || cost < best) { best = cost; *splits = s; }
  }
  return static_cast<int>(tiles);
}

}  // namespace sb

// fp32 elements of workspace that sb_paged_prefill needs; 0: none, `work` may be null.
extern "C" long sb_paged_prefill_workspace(int T, int B, int Hkv, int G, int P, int page, int D) {
  int splits;
  const long tiles = sb::paged_prefill_shape(T, B, Hkv, G, static_cast<long>(P) * page, &splits);
  return splits > 1 ? splits * tiles * Hkv * 256L * (D + 2) : 0;
}

// As sb_paged_attention, for any number of rows per sequence (max_rows is not read) and of query heads per kv head.
extern "C" int sb_paged_prefill(const sb::PagedAttentionArgs* args) {
  using namespace sb;
  SB_CHECK_ARG(args != nullptr);
  const PagedAttentionArgs& c = *args;
  const int shift = page_shift_of(c.page);
  SB_CHECK_ARG((c.D == 64 || c.D == 128) && shift >= 0 && c.Hq > 0 && c.Hkv > 0 && c.Hq % c.Hkv == 0 && c.T > 0 && c.B > 0 && c.P > 0 && c.num_pages > 0);
  SB_CHECK_ARG((c.starts != nullptr || c.T == c.B) && (c.k_scale == nullptr) == (c.v_scale == nullptr) && c.scale > 0.f);
  SB_CHECK_ARG(aligned16(c.q, c.k, c.v, c.o, c.work) && (c.q_ld | c.q_head | c.o_ld | c.o_head) % 8 == 0);
  SB_CHECK_ARG(static_cast<long>(c.T) * c.Hq < (1L << 31) - 256);
  const bool fp8 = c.k_scale != nullptr;
  const long size = fp8 ? 1 : 2;
  SB_CHECK_ARG(c.k_page >= 0 && c.v_page >= 0 && c.k_head >= 0 && c.v_head >= 0 && c.k_page * size < (1L << 32) && c.v_page * size < (1L << 32));
  PagedPrefillParams p;
  p.batch = PagedBatch{c.table, c.lengths, c.starts, c.table_ld, c.P, c.B, c.T, c.T, shift, c.num_pages};
  p.q = static_cast<const __nv_bfloat16*>(c.q); p.q_ld = c.q_ld; p.q_head = c.q_head;
  p.o = static_cast<__nv_bfloat16*>(c.o); p.o_ld = c.o_ld; p.o_head = c.o_head;
  p.k = static_cast<const uint8_t*>(c.k); p.v = static_cast<const uint8_t*>(c.v);
  p.k_page = c.k_page * size; p.k_head = c.k_head * size; p.v_page = c.v_page * size; p.v_head = c.v_head * size;
  p.ks = c.k_scale; p.vs = c.v_scale; p.ks_ld = c.k_scale_ld; p.vs_ld = c.v_scale_ld;
  p.Hq = c.Hq; p.Hkv = c.Hkv; p.G = c.Hq / c.Hkv;
  p.causal = c.causal; p.window = c.window; p.scale_log2 = c.scale * 1.4426950408889634f;
  p.zero_tail = c.zero_tail; p.part = c.work;
  p.tiles = paged_prefill_shape(c.T, c.B, c.Hkv, p.G, static_cast<long>(c.P) * c.page, &p.splits);
  SB_CHECK_ARG(p.tiles <= 65535 && (p.splits == 1 || c.work != nullptr));
  p.err = error_word();
  if (!p.err) return SB_ERR_CUDA;
  if (c.D == 64) return fp8 ? launch_paged_prefill<64, true>(p, c.stream) : launch_paged_prefill<64, false>(p, c.stream);
  return fp8 ? launch_paged_prefill<128, true>(p, c.stream) : launch_paged_prefill<128, false>(p, c.stream);
}
