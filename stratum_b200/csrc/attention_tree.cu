// Attention of drafted tokens over the paged cache: every sequence brings a tree of tokens, each of which sees the cached
// keys in front of the tree and its own ancestors in it.
//
// For query head h of drafted token i of a sequence with `base` cached keys: score_t = (q_h . K_t[kv(h)]) * scale over the
// cached keys t < base (with a window W: t > pos_i - W) and the drafted keys t = base + j with bit j of mask_i set;
// p = softmax, o_h = sum_t p_t V_t[kv(h)]; a row that sees no key gives zeros.  The drafted tokens' own keys and values lie
// in the cache already, row j at position base + j, in the order of the batch.
//
// A row of work is (token, head of the group); the rows of a sequence and a kv head share its keys, so the time to beat
// is one pass over the live pages.  As in attention_stream.cu the pages of all (sequence, kv head, tile of rows) form one
// list of units, CTA c takes the stretch [c T / G, (c + 1) T / G), and what several CTAs saw pieces of is added up by
// attention_tree_merge_kernel, in CTA order.  Everything the cut depends on is read from the device, so a captured launch
// serves whatever lengths the description holds at its replay.
//
// Two kernels.  attention_tree_tc_kernel: bfloat16, heads of 64 or 128, on tcgen05 (below).  attention_tree_simple_kernel:
// any head size up to 256, float32 or bfloat16, on the CUDA cores in float32 throughout.
//
// The tcgen05 kernel.  A CTA has two halves, each with a warp that issues MMAs, four softmax warps (a thread per row),
// two buffers of scores and an accumulator in tensor memory: S = Q K^T (128 rows x 64 keys), P = exp(S - ref), O += P V.
//   ROWS2 = false (at most 128 rows per sequence and kv head): both halves hold the same rows and take every other page,
//     so that one page's softmax runs under the other's loads and MMAs; their sums are joined at the end of a run;
//   ROWS2 = true: the halves hold 128 rows each and share every page, which then is fetched once for 256 rows.
// P goes back into tensor memory, over the scores it came from, and is the first operand of P V there: with P in shared
// memory its writing and its reading by the MMAs took a third of what shared memory moves per tile, and every tile had to
// wait for the one before to be read (91 us against 83 for one sequence of 32,700 tokens and 61 drafted ones).
// One thread of warp 0 feeds rings of K and V pages by TMA, and the queries of the run that comes next; the last warp walks the
// list ahead of the others.
//
// The products with masked keys: P is zero there, but zero times an infinity or a NaN is not, and a page that is masked for
// some row may hold either (rows behind the sequence's end, a drafted branch that overflowed).  So the V page of a masked
// tile is looked through, by the last warp as soon as it is there; rows of V that are not finite are zeroed in shared memory, and
// what they give to the rows that do see them is added by hand.
//
// Every mbarrier wait is bounded: on expiry a code goes to the status word and a flag is set that ends every other wait of
// the block, so that all leave together.
//
// What bounds the tcgen05 kernel.  64 keys of 256 rows take 2,000 to 2,200 cycles, of which the tensor cores are busy for
// 1,270 (a product of 128 x 64 x 16 takes them 48 cycles with both halves at it, as the rows of Q are read from shared memory
// each time, one of 128 x 128 x 16 takes 64) and the exponentials' units for 1,024; the rest is one waiting for the other
// at the ends of tiles.  Around the tiles: 3 us to read the list, 3 more to the first scores, 3 at the end of a run (the last
// product, the outputs), 6 to add pieces up.  Measured, 8 kv heads of 4 queries, head size 128, calls one behind the other:
// one sequence of 32,700 tokens and 61 drafted ones 58 us (134 MB of keys and values, 2.3 TB/s, 560 TFLOP/s; 54 in a replayed graph of
// ten calls); 64 sequences of 4,000 and 33 to 64 drafted ones 315 (3.1 TB/s, 565 TFLOP/s: the card is at its power limit; 267 in
// the graph, before it gets there).
// Tried without a gain: more of the exponentials as polynomials, a lock that keeps the halves' products apart, halves that start
// half a tile apart, one thread that issues for both, a guess at the maximum before the scores are there.
#include <math.h>

#include "tc_common.cuh"

#define TR_KEYS 64
#define TR_MAX_SEQS 4096
#define TR_SOFTMAX_WARPS 4                  // per half, a thread a row
#define TR_THREADS (32 + 2 * 32 + 2 * TR_SOFTMAX_WARPS * 32 + 32)
#define TR_RUNS 4
#define TR_LOOKS 16

struct TreeParams {
  const int* token_pos;                    // [tokens]
  const unsigned long long* mask; int words;   // [tokens][words]
  const int* seq_start; const int* seq_len;    // [seqs + 1], [seqs]
  const int* block_table; int bt_stride, bt_width;
  const void* q; int ldq;
  const void* k_cache; const void* v_cache;
  void* out; int ldo;
  float4* part_o;                          // [G][2][head_dim / 4][rows of a slot]: pieces, unnormalised (a warp has rows)
  float2* part_ml;                         // [G][2][rows per tile]: their (maximum, sum)
  struct TreeCut* cut;                     // [G]: what each CTA's stretch begins in
  int* status;
  int n_tokens, n_seqs, n_q, n_kv, gs, head_dim, window, n_pages, rows_per_tile;
  int item_units;                          // (see the list of units)
  int out_by_16;                           // a head's row of the output begins on 16 bytes and is a multiple of them
  float scale;
};

// The cut in front of CTA c's stretch, for the merge.
struct alignas(16) TreeCut {
  int first, cuts;                         // the CTA that has the item's first page, how many cuts go through the item (0: this one
                                           // goes through none)
  int late, kvh;                           // whether that CTA's stretch begins in front of the item; the item's kv head,
  int flat0, n_rows;                       // its first row (token of the batch * gs + head), its rows
  int pad[2];
};
static_assert(sizeof(TreeCut) == 32, "as the launcher lays them out");

struct TreeSeq {                           // a sequence's share of the list
  int row0, n_new, base, len, first, n_pages, n_tiles, tile_rows;
  int w, units;                            // units of a page (on the CUDA cores: else one), of an item
};
// CORES: for the CUDA cores, where time goes by rows: a tree's rows are shared out evenly among its tiles (68 as 40 and 28, not
// as 64 and 4), and a page weighs as many units as a thread has rows of it, and two.
template <bool CORES>
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& P, int b) {
  TreeSeq s;
  s.row0 = min(max(__ldcg(P.seq_start + b), 0), P.n_tokens);
  s.n_new = min(max(__ldcg(P.seq_start + b + 1), s.row0), P.n_tokens) - s.row0;
  s.len = max(__ldcg(P.seq_len + b), 0);
  s.base = max(s.len - s.n_new, 0);
  const int pages = max(min((int)(((long long)s.len + TR_KEYS - 1) / TR_KEYS), P.bt_width), 1);
  const int lo = (P.window > 0 && s.base - P.window + 1 > 0) ? s.base - P.window + 1 : 0;
  s.first = min(lo / TR_KEYS, pages - 1);
  s.n_pages = pages - s.first;
  const int rows = s.n_new * P.gs;
  s.n_tiles = (rows + P.rows_per_tile - 1) / P.rows_per_tile;
  s.tile_rows = CORES && s.n_tiles > 1 ? ((rows + s.n_tiles - 1) / s.n_tiles + 7) & ~7 : P.rows_per_tile;
  s.w = CORES ? ((min(rows, s.tile_rows) + 15) >> 4) + 2 : 1;
  s.units = s.w * s.n_pages + P.item_units;
  return s;
}
// The list of units: every item (sequence, kv head, tile of rows) has those of its pages (one each on the tensor cores) and a few
// more behind them, for what an item costs besides its pages (on the tensor cores: its masked pages, its outputs, and the next
// item's first scores).  A page is the CTA's whose stretch its first unit lies in.  Without the few more a CTA whose stretch was made
// of short sequences took 80 us where the others took 46; with 3 instead of 7 on the tensor cores 24 sequences took 58 us instead
// of 53; with pages of one unit on the CUDA cores, whatever their rows, five sequences took 62 instead of 56.  A short list is cut
// among fewer CTAs, TREE_LEAST_UNITS to each (three times as many on the CUDA cores): what a piece of one page saves in its own
// time, adding up its pieces costs again.  No stretch is then shorter than a page's units (at most 6, and a list of more than 12
// (n - 1) units is cut among n CTAs, n > 1: 6 each at least), so every stretch that begins in front of an item's last page has a
// page of it.
#define TREE_LEAST_UNITS 4
template <bool CORES>
__device__ __forceinline__ int tree_ctas(long long T, int G) {
  const int least = CORES ? 3 * TREE_LEAST_UNITS : TREE_LEAST_UNITS;
  const long long n = (T + least - 1) / least;
  return n < 1 ? 1 : n < G ? (int)n : G;
}
__device__ __forceinline__ long long tree_begin(int c, int ctas, long long T) { return c >= ctas ? T : (long long)c * T / ctas; }

// A stretch of pages of one item.
struct TreeRun {
  TreeSeq s;
  int b, kvh, rt, page0, n;                // n = 0: there are no more
  int clean0, clean1;                      // of its pages, those that every row sees whole; the others are masked
  bool from_start, to_end, holds_u0;
  bool pages_ok;                           // no page lies outside the pool
};

template <bool CORES>
struct TreeCursor {
  int left;                                // units of the stretch that are still ahead
  int b, item, off;
  bool moved;
  TreeSeq s;
  __device__ __forceinline__ void step(const TreeParams& P, int n) {
    moved = true;
    off += n; left -= n;
    if (off < s.units) return;
    off = 0;
    if (++item < s.n_tiles * P.n_kv) return;
    item = 0;
    do { b++; if (b < P.n_seqs) s = tree_seq<CORES>(P, b); } while (b < P.n_seqs && s.n_tiles == 0);
  }
  __device__ __forceinline__ void next(const TreeParams& P, TreeRun& r) {
    int p0 = 0, n = 0;
    while (left > 0) {
      const int w = CORES ? s.w : 1;
      p0 = (off + w - 1) / w;                    // the first page that begins in the stretch, and how many do
      n = min((off + left + w - 1) / w, s.n_pages) - p0;
      if (n > 0) break;
      step(P, min(s.units - off, left));
    }
    if (left <= 0) { r.n = 0; return; }
    r.s = s; r.b = b;
    r.kvh = item / s.n_tiles; r.rt = item % s.n_tiles;
    r.page0 = s.first + p0;
    r.n = n;
    r.from_start = p0 == 0;
    r.to_end = p0 + n == s.n_pages;
    r.holds_u0 = !moved;
    step(P, min(s.units - off, left));
  }
};

// Where CTA c begins; every thread of the block calls it.  `sums` holds a running sum per sequence for the while.
template <bool CORES>
__device__ __forceinline__ TreeCursor<CORES> tree_start(const TreeParams& P, long long* sums, long long& u0_, long long& total_) {
  const int n_threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b < P.n_seqs; b += n_threads) {
    const TreeSeq s = tree_seq<CORES>(P, b);
    sums[b + 1] = (long long)s.units * s.n_tiles * P.n_kv;
  }
  if (threadIdx.x == 0) sums[0] = 0;
  __syncthreads();
  if (warp == 0) {
    long long carry = 0;
    for (int base = 0; base < P.n_seqs; base += 32) {
      const int i = base + lane;
      long long v = i < P.n_seqs ? sums[i + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += n;
      }
      if (i < P.n_seqs) sums[i + 1] = v + carry;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  TreeCursor<CORES> t;
  const long long T = sums[P.n_seqs];
  const int c = blockIdx.x, ctas = tree_ctas<CORES>(T, gridDim.x);
  const long long u0 = tree_begin(c, ctas, T);
  t.left = (int)(tree_begin(c + 1, ctas, T) - u0);
  t.b = t.item = t.off = 0;
  t.moved = false;
  u0_ = u0; total_ = T;
  if (t.left > 0) {
    int lo = 0, hi = P.n_seqs - 1;                // the last sequence that begins at or before u0 and is not empty
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sums[mid] <= u0) lo = mid; else hi = mid - 1;
    }
    t.s = tree_seq<CORES>(P, lo);
    const long long r = u0 - sums[lo];
    const int per = t.s.units;
    t.b = lo; t.item = (int)(r / per); t.off = (int)(r % per);
  }
  return t;
}
// The last CTA whose stretch begins at or before unit u (0 <= u < T).
__device__ __forceinline__ int tree_cta_of(long long u, int ctas, long long T) {
  int c = min((int)(u * ctas / T), ctas - 1);      // floor(c T / ctas) <= u, and at most one short
  while (c + 1 < ctas && tree_begin(c + 1, ctas, T) <= u) c++;
  return c;
}
// One thread, with the cursor as tree_start left it: what the merge is to know about the cut in front of this stretch.
template <bool CORES>
__device__ __forceinline__ void tree_cut(const TreeParams& P, const TreeCursor<CORES>& t, long long u0, long long T) {
  TreeCut cut;
  cut.first = cut.cuts = cut.late = cut.kvh = cut.flat0 = cut.n_rows = 0;
  const int last = (CORES ? t.s.w : 1) * (t.s.n_pages - 1);      // where the item's last page begins
  if (t.left > 0 && t.off > 0 && t.off <= last) {
    const long long begin = u0 - t.off;
    const int ctas = tree_ctas<CORES>(T, gridDim.x), rt = t.item % t.s.n_tiles;
    cut.first = tree_cta_of(begin, ctas, T);
    cut.cuts = tree_cta_of(begin + last, ctas, T) - cut.first;
    cut.late = tree_begin(cut.first, ctas, T) != begin;
    cut.kvh = t.item / t.s.n_tiles;
    cut.flat0 = t.s.row0 * P.gs + rt * t.s.tile_rows;
    cut.n_rows = min(t.s.n_new * P.gs - rt * t.s.tile_rows, t.s.tile_rows);
  }
  P.cut[blockIdx.x] = cut;
}

// Which of the 64 keys from position `key0` on a drafted token sees; word0: the first word of its mask.
__device__ __forceinline__ unsigned long long tree_visible(const TreeParams& P, const TreeSeq& s, int token, int lo, int key0,
                                                           bool page_ok, unsigned long long word0) {
  if (!page_ok) return 0;
  const unsigned long long all = ~0ull;
  unsigned long long cached = 0;
  const int to_base = s.base - key0;               // cached keys from here on
  if (to_base >= 64) cached = all;
  else if (to_base > 0) cached = (1ull << to_base) - 1;
  const int to_lo = lo - key0;
  if (to_lo >= 64) cached = 0;
  else if (to_lo > 0) cached &= all << to_lo;
  unsigned long long nodes = 0;
  if (to_base < 64) {                              // drafted keys in this page: node 0 lies at bit to_base
    const unsigned long long* m = P.mask + (size_t)token * P.words;
    const int n = min(s.n_new, 64 * P.words);
    auto word = [&](int w) -> unsigned long long {
      if (64 * w >= n) return 0;
      const unsigned long long v = w == 0 ? word0 : __ldcg(m + w);
      return n - 64 * w >= 64 ? v : v & ((1ull << (n - 64 * w)) - 1);
    };
    if (to_base > 0) nodes = word(0) << to_base;
    else {
      const int o = -to_base, w = o >> 6, sh = o & 63;
      nodes = word(w) >> sh;
      if (sh) nodes |= word(w + 1) << (64 - sh);
    }
  }
  unsigned long long v = cached | nodes;
  const int left = s.len - key0;                   // nothing behind the sequence's end
  if (left < 64) v &= left > 0 ? (1ull << left) - 1 : 0;
  return v;
}

// ================================================================ tcgen05
template <int HD, bool ROWS2>
struct TreeSmem {
  static constexpr int STAGES = HD == 64 ? 10 : ROWS2 ? 5 : 4;   // (even where the halves alternate: a stage is then always the same half's)
  static constexpr int QB = ROWS2 ? 1 : 2;              // queries of the next run beside those of this one
  alignas(1024) bf16 q[2][128 * HD];                    // ROWS2: per half; else: of two runs
  alignas(1024) bf16 k[STAGES][TR_KEYS * HD];           // [HD/64][64 keys][64 dims]
  alignas(1024) bf16 v[STAGES][TR_KEYS * HD];
  float2 ml[2][ROWS2 ? 1 : 128];                                    // a row's maximum and sum in either half, at the end of a run
  uint64_t q_full[QB], q_empty[QB], k_full[STAGES], v_full[STAGES];
  uint64_t s_full[2][STAGES], pv_full[2][STAGES], p_full[2][2];
  unsigned long long bad[2][TR_LOOKS];                  // per half (ROWS2: for both), of its masked tiles in turn: keys with values not finite
  uint64_t look_full[2][TR_LOOKS];
  uint32_t v_asked;                                     // tiles whose values have been asked for
  TreeRun runs[TR_RUNS];                                // the runs ahead, from the warp that walks the list
  uint64_t run_full[TR_RUNS], run_seen[TR_RUNS], run_empty[TR_RUNS];     // (seen: what only the softmax warps ask for is there too)
  uint64_t run_meet;                                    // softmax warps wait for one another (bounded, as every wait)
  int row_of[32];                                       // cache row of a tile's page, from the K to the V request
  uint32_t tmem_base;
  int o_ready[2];
  int abort_flag;
};

__device__ __forceinline__ float tr_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two floats in a register pair: an instruction does both (what the softmax threads have too many of is instructions)
__device__ __forceinline__ uint64_t tr_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void tr_split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t tr_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t tr_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t tr_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float tr_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^a and 2^b with additions and products alone (a and b below 2^7): the whole part n goes into a float's exponent, 2^f of the
// rest, |f| <= 1/2, is a cubic, fitted to the smallest largest relative error there, 7.5e-5 (2^-13.7: what is rounded to bfloat16 does
// not notice).  0 below 2^-126; no number stays none.
__device__ __forceinline__ void tr_exp2_pair(float& a, float& b) {
  float x0, x1, t0, t1;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(a), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(b), "f"(-127.f));
  const uint64_t x = tr_pair(x0, x1);
  const float shift = 12582912.f + 127.f;                // 1.5 * 2^23: behind it the last bits hold n + 127
  const uint64_t t = tr_add2(x, tr_pair(shift, shift));
  const uint64_t f = tr_fma2(tr_add2(t, tr_pair(-shift, -shift)), tr_pair(-1.f, -1.f), x);
  uint64_t p = tr_fma2(f, tr_pair(0.05517167f, 0.05517167f), tr_pair(0.24261113f, 0.24261113f));
  p = tr_fma2(p, f, tr_pair(0.69326097f, 0.69326097f));
  p = tr_fma2(p, f, tr_pair(0.99992806f, 0.99992806f));
  tr_split(t, t0, t1);
  const uint64_t power = tr_pair(__uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23));
  tr_split(tr_mul2(p, power), a, b);
}
// The warps that `bar` counts wait for one another: false if one of them has given up.
__device__ __forceinline__ bool tr_meet(uint64_t* bar, uint32_t phase, volatile int* abort_flag) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag));
}
// two outputs as bfloat16; zeros where the row's sum L is zero (it saw no key)
__device__ __forceinline__ uint32_t tr_pack(float L, float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(L == 0.f ? 0.f : a, L == 0.f ? 0.f : b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Four lanes hold 64 bytes of a row each: behind this each has 16 bytes of all four rows, w[k] of the k-th, so that what a store
// writes lies together (a row a lane, every store touched 32 lines, and a run's outputs took 4 us).
__device__ __forceinline__ void tr_turn(uint4 (&w)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int x = 1; x < 4; x *= 2)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (k & x) continue;
      uint4 give = lane & x ? w[k] : w[k + x];
      give.x = __shfl_xor_sync(0xffffffffu, give.x, x); give.y = __shfl_xor_sync(0xffffffffu, give.y, x);
      give.z = __shfl_xor_sync(0xffffffffu, give.z, x); give.w = __shfl_xor_sync(0xffffffffu, give.w, x);
      if (lane & x) w[k] = give; else w[k + x] = give;
    }
}
__device__ __forceinline__ float tmem_ld1f(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  tmem_ld_wait();
  return __uint_as_float(r);
}

__device__ __forceinline__ void tr_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// D += A B with A (128 rows x 16 bfloat16) in tensor memory: two values of k to a column
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

#define TR_FAIL(code) { atomicCAS(P.status, 0, code); S.abort_flag = 1; }

// What only masked tiles need is functions of their own, so that the loop over the other tiles keeps its registers.

// The keys of a page of values (in shared memory) that hold anything not finite; their rows are zeroed.  One warp, two keys a
// lane.
template <int HD>
__device__ __noinline__ unsigned long long tree_look_through(uint4* v) {
  const int lane = threadIdx.x & 31;
  uint32_t most[2] = {0, 0};                             // largest magnitude, as two numbers of 15 bits
  // 8 chunks of 16 bytes a key and block of 64 dims, visited from another one on by each key: all banks
  auto chunk = [&](int c, int key) { return v + key * 8 + (c >> 3) * (TR_KEYS * 8) + ((c + key) & 7); };
#pragma unroll 4
  for (int c = 0; c < HD / 8; c++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const uint4 x = *chunk(c, lane + 32 * e);
      most[e] = __vmaxu2(__vmaxu2(most[e], x.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(x.y & 0x7fff7fffu, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu));
    }
  bool odd[2];
#pragma unroll
  for (int e = 0; e < 2; e++) odd[e] = (most[e] & 0xffffu) >= 0x7f80u || (most[e] >> 16) >= 0x7f80u;
  const unsigned long long bad = __ballot_sync(0xffffffffu, odd[0]) | (unsigned long long)__ballot_sync(0xffffffffu, odd[1]) << 32;
  if (bad) {
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (odd[e])
        for (int c = 0; c < HD / 8; c++) *chunk(c, lane + 32 * e) = make_uint4(0, 0, 0, 0);
    fence_async_shared();
    __syncwarp();
  }
  return bad;
}

// A weight is 2^(score to_log2 - m_ref) with one rounding.  m_ref is a rounded product itself, so that all weights of a row have a
// factor in common, which their sum takes out again: 2^64 at most for references below TR_LARGE, without end above.  There the
// score's product is rounded too, as m_ref was, and the largest weight is one.
#define TR_LARGE 0x1p30f
__device__ __forceinline__ float tree_weight(float score, float to_log2, float m_use) {
  return tr_exp2(fabsf(m_use) >= TR_LARGE ? __fmul_rn(score, to_log2) - m_use : fmaf(score, to_log2, -m_use));
}

// P of a tile of a warp that has rows of such scores, over the scores (the first half's end where the second half's begin); the sum
// of this thread's row.
__device__ __noinline__ float tree_large_scores(unsigned long long vis, uint32_t s_addr, float to_log2, float m_use) {
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < TR_KEYS; c += 32) {
    uint32_t r[32], packed[16];
    tmem_ld32(s_addr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float p0 = (vis >> (c + e)) & 1 ? tree_weight(__uint_as_float(r[e]), to_log2, m_use) : 0.f;
      const float p1 = (vis >> (c + e + 1)) & 1 ? tree_weight(__uint_as_float(r[e + 1]), to_log2, m_use) : 0.f;
      uint32_t u;
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(p1), "f"(p0));
      sum += __uint_as_float(u << 16) + __uint_as_float(u & 0xffff0000u);
      packed[e >> 1] = u;
    }
    tr_store16(s_addr + c / 2, packed);
  }
  return sum;
}

// Adds what the keys in `bad` give to this thread's row of the output in tensor memory (or to zeros where it holds nothing
// yet).  v: the page's values in the cache.
template <int HD>
__device__ __noinline__ void tree_add_bad(unsigned long long bad, unsigned long long vis, uint32_t s_addr, uint32_t o_addr,
                                          float to_log2, float m_use, const bf16* v, bool fresh) {
  for (int c = 0; c < HD; c += 32) {
    uint32_t r[32];
    tmem_ld32(o_addr + c, r);
    tmem_ld_wait();
    if (fresh) {
#pragma unroll
      for (int e = 0; e < 32; e++) r[e] = 0;
    }
    for (int k = 0; k < 64; k++) {
      if (!((bad >> k) & 1)) continue;
      const float p = tree_weight(tmem_ld1f(s_addr + k), to_log2, m_use);
      const bool sees = (vis >> k) & 1;
#pragma unroll
      for (int e = 0; e < 32; e++)
        if (sees) r[e] = __float_as_uint(fmaf(p, ld_fresh(v + (size_t)k * HD + c + e), __uint_as_float(r[e])));
    }
    tmem_st32(o_addr + c, r);
  }
  tmem_st_wait();
}

template <int HD, bool ROWS2>
__global__ void __launch_bounds__(TR_THREADS, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const TreeParams P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  using Smem = TreeSmem<HD, ROWS2>;
  constexpr int STAGES = Smem::STAGES, QB = Smem::QB, DB = HD / 64;
  constexpr uint32_t COL_PV = 128;
  static_assert(sizeof(Smem) <= 227 * 1024, "shared memory of an SM");
  static_assert(STAGES < TR_LOOKS, "a masked tile's entry is read before the tile that has it next is there");
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023) {                      // (the swizzled tiles need it)
    if (threadIdx.x == 0) {
      atomicCAS(P.status, 0, 510);
      P.cut[blockIdx.x] = TreeCut{};
    }
    return;
  }
  volatile int* abort_flag = &S.abort_flag;
  if (threadIdx.x == 0) {
    for (int i = 0; i < QB; i++) { mbar_init(&S.q_full[i], 1); mbar_init(&S.q_empty[i], 2); }
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&S.k_full[s], 1); mbar_init(&S.v_full[s], 1);
      for (int h = 0; h < 2; h++) { mbar_init(&S.s_full[h][s], 1); mbar_init(&S.pv_full[h][s], 1); }
    }
    for (int h = 0; h < 2; h++) {
      mbar_init(&S.p_full[h][0], TR_SOFTMAX_WARPS); mbar_init(&S.p_full[h][1], TR_SOFTMAX_WARPS);
      S.o_ready[h] = 0;
      for (int i = 0; i < TR_LOOKS; i++) mbar_init(&S.look_full[h][i], 1);
    }
    for (int i = 0; i < TR_RUNS; i++) { mbar_init(&S.run_full[i], 1); mbar_init(&S.run_seen[i], 1); mbar_init(&S.run_empty[i], 4 + 2 * TR_SOFTMAX_WARPS); }
    S.v_asked = 0;
    mbar_init(&S.run_meet, 2 * TR_SOFTMAX_WARPS);
    S.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(&S.tmem_base, 512);
    tmem_relinquish();
  }
  pdl_wait();                                           // everything below may read what the kernel before this one wrote
  long long u0, total;
  TreeCursor<false> cur = tree_start<false>(P, reinterpret_cast<long long*>(S.k), u0, total);
  fence_async_shared();                                 // the sums lie where TMA will write
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = S.tmem_base;
  const int gs = P.gs;
  const int half_tokens = 128 / gs;                     // tokens of a half's 128 rows
  auto half_ntok = [&](const TreeRun& r, int h) {       // tokens of the run's tile that half h holds
    const int t0 = ROWS2 ? (2 * r.rt + h) * half_tokens : r.rt * half_tokens;
    return min(max(r.s.n_new - t0, 0), half_tokens);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
      // runs whose queries, whose keys have been asked for, whose place in the ring has been given back
      int nq = 0, nr = 0, given = 0;
      bool more_q = true, more_k = true, in_run = false;
      int tile = 0, pg = 0;
      uint32_t jk = 0, jv = 0;
      auto freed = [&](uint64_t (*bars)[STAGES], uint32_t j) -> bool {   // tile j - STAGES has been read
        const uint32_t par = ((j / STAGES) - 1) & 1;
        if (ROWS2) return mbar_test_wait(&bars[0][j % STAGES], par) && mbar_test_wait(&bars[1][j % STAGES], par);
        return mbar_test_wait(&bars[j & 1][j % STAGES], par);
      };
      uint32_t idle = 0;
      bool ok = true;
      while ((more_q || more_k || jv < jk) && ok) {
        bool moved = false;
        if (more_q && mbar_test_wait(&S.run_full[nq % TR_RUNS], (nq / TR_RUNS) & 1)) {
          const TreeRun& rq = S.runs[nq % TR_RUNS];
          if (rq.n == 0) {
            more_q = false;
            moved = true;
          } else if (nq < QB || mbar_test_wait(&S.q_empty[nq % QB], ((nq / QB) - 1) & 1)) {
            uint64_t* bar = &S.q_full[nq % QB];
            const uint32_t box = (uint32_t)half_tokens * gs * HD * sizeof(bf16);
            const bool second = ROWS2 && half_ntok(rq, 1) > 0;
            mbar_expect_tx(bar, second ? 2 * box : box);
            const int tok0 = rq.s.row0 + rq.rt * half_tokens * (ROWS2 ? 2 : 1);
            for (int db = 0; db < DB; db++) {
              tma_load_3d(&map_q, S.q[ROWS2 ? 0 : nq % QB] + db * 128 * 64, bar, db * 64, rq.kvh * gs, tok0);
              if (second) tma_load_3d(&map_q, S.q[1] + db * 128 * 64, bar, db * 64, rq.kvh * gs, tok0 + half_tokens);
            }
            nq++;
            moved = true;
          }
        }
        if (more_k && !in_run && mbar_test_wait(&S.run_full[nr % TR_RUNS], (nr / TR_RUNS) & 1)) {
          const TreeRun& run = S.runs[nr % TR_RUNS];
          if (run.n == 0) more_k = false;
          else {
            in_run = true; tile = 0;
            pg = __ldcg(P.block_table + (size_t)run.b * P.bt_stride + run.page0);
          }
          moved = true;
        }
        if (in_run && (jk < STAGES || freed(S.s_full, jk))) {
          const TreeRun& run = S.runs[nr % TR_RUNS];
          const int s = jk % STAGES;
          // (a page number outside the pool: some page's rows are fetched and nobody sees them)
          const int row = (int)(((long long)((unsigned)pg < (unsigned)P.n_pages ? pg : 0) * P.n_kv + run.kvh) * TR_KEYS);
          S.row_of[jk & 31] = row;
          mbar_expect_tx(&S.k_full[s], TR_KEYS * HD * sizeof(bf16));
          for (int db = 0; db < DB; db++) tma_load_2d(&map_k, S.k[s] + db * TR_KEYS * 64, &S.k_full[s], db * 64, row);
          jk++;
          if (++tile == run.n) { in_run = false; nr++; }
          else pg = __ldcg(P.block_table + (size_t)run.b * P.bt_stride + run.page0 + tile);
          moved = true;
        }
        if (given < nq && given < nr) { mbar_arrive(&S.run_empty[given % TR_RUNS]); given++; }
        if (jv < jk && (jv < STAGES || freed(S.pv_full, jv))) {
          const int s = jv % STAGES, row = S.row_of[jv & 31];
          mbar_expect_tx(&S.v_full[s], TR_KEYS * HD * sizeof(bf16));
          for (int db = 0; db < DB; db++) tma_load_2d(&map_v, S.v[s] + db * TR_KEYS * 64, &S.v_full[s], db * 64, row);
          jv++;
          *(volatile uint32_t*)&S.v_asked = jv;
          moved = true;
        }
        if (moved) { idle = 0; continue; }
        __nanosleep(32);
        if (++idle >= 4u * TC_SPIN_LIMIT || ((idle & 1023u) == 0 && *abort_flag)) { TR_FAIL(501); ok = false; }
      }
      pdl_trigger();
      if (!ok) {
        for (int i = 0; i < 2000; i++) __nanosleep(1000);   // let copies already issued land
      }
    }
  } else if (warp <= 2) {
    // ---------------------------------------------------------------- MMA issuer of half `warp - 1`
    const int h = warp - 1;
    const uint32_t idesc_s = instr_desc_bf16(TR_KEYS), idesc_pv = instr_desc_bf16(HD, true);
    const uint32_t tmem_h = tmem_base + h * 256;
    bool ok = true;
    // This half's tiles as one sequence over the runs, the scores one tile ahead of the products with V: what is known of
    // the tile whose P V is still to come
    bool pend = false, pend_first = false, pend_active = false;
    uint32_t pend_it = 0, pend_i = 0;
    uint32_t it = 0, i = 0;                              // tiles of the stretch, of this half
    auto values = [&]() {                                // P V of the pending tile
      const int s = pend_it % STAGES;
      if (!__all_sync(0xffffffffu, mbar_wait(&S.v_full[s], (pend_it / STAGES) & 1, abort_flag))) { if (lane == 0) TR_FAIL(506); ok = false; return; }
      if (!__all_sync(0xffffffffu, mbar_wait(&S.p_full[h][pend_i & 1], (pend_i >> 1) & 1, abort_flag))) { if (lane == 0) TR_FAIL(505); ok = false; return; }
      if (!pend_active) {                                // no rows of this half: the page is free
        if (lane == 0) mbar_arrive(&S.pv_full[h][s]);
        __syncwarp();
        return;
      }
      tc_fence_after();
      const uint64_t vd = smem_desc_sw128_mn(smem_u32(S.v[s]), TR_KEYS * 128);
      const uint32_t p_addr = tmem_h + (pend_i & 1) * TR_KEYS;
      const bool fresh = pend_first && *(volatile int*)&S.o_ready[h] == 0;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; kk++)                   // 16 keys a step: 8 columns of P, 16 rows of V (in units of 16 bytes)
          umma_bf16_ts(tmem_h + COL_PV, p_addr + kk * 8, vd + (uint64_t)(kk * 16 * 128 / 16), idesc_pv, (fresh && kk == 0) ? 0u : 1u);
        umma_commit(&S.pv_full[h][s]);
      }
      __syncwarp();
    };
    // ROWS2, whose next queries come once this run's scores are through: until they are here, the product that the softmax warps
    // need to end this run (with the halves in turn on one tile the queries are there already)
    auto or_values = [&](uint64_t* bar, uint32_t parity) {
      if (ROWS2 && pend && !__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) { values(); pend = false; }
    };
    for (int r = 0; ok; r++) {
      or_values(&S.run_full[r % TR_RUNS], (r / TR_RUNS) & 1);
      if (!ok) break;
      if (!__all_sync(0xffffffffu, mbar_wait(&S.run_full[r % TR_RUNS], (r / TR_RUNS) & 1, abort_flag))) { if (lane == 0) TR_FAIL(511); ok = false; break; }
      const TreeRun& run = S.runs[r % TR_RUNS];
      if (run.n == 0) break;
      const bool active = !ROWS2 || half_ntok(run, h) > 0;
      or_values(&S.q_full[r % QB], (r / QB) & 1);
      if (!ok) break;
      if (!__all_sync(0xffffffffu, mbar_wait(&S.q_full[r % QB], (r / QB) & 1, abort_flag))) { if (lane == 0) TR_FAIL(502); ok = false; break; }
      const uint64_t qd = smem_desc_sw128(smem_u32(S.q[ROWS2 ? h : r % QB]));
      bool first = true;
      const uint32_t it_end = it + run.n;
      for (; it < it_end && ok; it++) {
        if (!ROWS2 && (int)(it & 1) != h) continue;
        const int s = it % STAGES;
        const uint32_t before2 = it - 2 * (ROWS2 ? 1 : 2);
        if (!__all_sync(0xffffffffu, mbar_wait(&S.k_full[s], (it / STAGES) & 1, abort_flag))) { if (lane == 0) TR_FAIL(503); ok = false; break; }
        if (active) {
          // the buffer holds P of two tiles ago: its product with V has been issued, and is over
          if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(&S.pv_full[h][before2 % STAGES], (before2 / STAGES) & 1, abort_flag))) { if (lane == 0) TR_FAIL(504); ok = false; break; }
          tc_fence_after();
          const uint64_t kd = smem_desc_sw128(smem_u32(S.k[s]));
          if (elect_one()) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
              for (int kk = 0; kk < 4; kk++)             // (descriptors count in units of 16 bytes)
                umma_bf16(tmem_h + (i & 1) * TR_KEYS, qd + (uint64_t)((db * 128 * 128 + kk * 32) / 16),
                          kd + (uint64_t)((db * TR_KEYS * 128 + kk * 32) / 16), idesc_s, (db | kk) ? 1u : 0u);
            umma_commit(&S.s_full[h][s]);
          }
          __syncwarp();
        } else {
          if (lane == 0) mbar_arrive(&S.s_full[h][s]);
          __syncwarp();
        }
        if (pend) values();
        pend = true; pend_first = first; pend_active = active; pend_it = it; pend_i = i;
        first = false;
        i++;
      }
      it = it_end;
      if (ok) {                                          // the run's scores are issued: its queries are free behind them
        if (elect_one()) umma_commit(&S.q_empty[r % QB]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.run_empty[r % TR_RUNS]);
      }
    }
    if (ok && pend) values();
  } else if (warp < 3 + 2 * TR_SOFTMAX_WARPS) {
    // ---------------------------------------------------------------- softmax (four warps per half, a thread a row)
    const int h = (warp - 3) / TR_SOFTMAX_WARPS;
    const int quarter = warp & 3;                        // tensor-memory lanes this warp may read
    const int row = quarter * 32 + lane;
    const int tok = row / gs, head = row % gs;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t lane_addr = lane_base + h * 256;
    const uint32_t o_addr = lane_addr + COL_PV;
    const float to_log2 = P.scale * 1.4426950408889634f;
    constexpr int STEP = ROWS2 ? 1 : 2;                  // from a tile of this half to the next
    bool ok = true;
    uint32_t it = 0, i = 0, run_phase = 0, looks = 0;    // tiles of the stretch, of this half, meetings, masked tiles of this half
#define TR_WAIT(bar, parity, code) \
  if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) { if (lane == 0) TR_FAIL(code); ok = false; break; }
    for (int r = 0; ok; r++) {
      TR_WAIT(&S.run_full[r % TR_RUNS], (r / TR_RUNS) & 1, 511)
      const TreeRun& run = S.runs[r % TR_RUNS];
      if (run.n == 0) break;
      const TreeSeq& sq = run.s;
      const int ntok = half_ntok(run, h);
      const bool valid = tok < ntok;
      const bool warp_active = quarter * 32 < ntok * gs;
      const int token = sq.row0 + (ROWS2 ? 2 * run.rt + h : run.rt) * half_tokens + (valid ? tok : 0);
      const int lo = (P.window > 0 && valid) ? max(__ldcg(P.token_pos + token) - P.window + 1, 0) : 0;
      const unsigned long long word0 = valid ? __ldcg(P.mask + (size_t)token * P.words) : 0;      // (for the last page or two)
      const uint32_t it_first = it, it_end = it + run.n;
      if (!ROWS2 && (int)(it & 1) != h) it++;
      const uint32_t it_mine = it;                       // this half's first tile of the run (it_end or beyond: none)
      const int* bt = P.block_table + (size_t)run.b * P.bt_stride + run.page0 - (int)it_first;   // [it]: the tile's page
      TR_WAIT(&S.run_seen[r % TR_RUNS], (r / TR_RUNS) & 1, 511)
      const uint32_t clean_from = it_first + run.clean0, clean_to = it_first + run.clean1;
      float m_ref = -INFINITY, l = 0.f;
      bool any_large = false;                            // some row of the warp has a reference beyond TR_LARGE
      for (; it < it_end; it += STEP) {
        const int s = it % STAGES, b = i & 1;
        const bool needs_mask = it < clean_from || it >= clean_to, first = it == it_mine;
        TR_WAIT(&S.s_full[h][s], (it / STAGES) & 1, 509)
        unsigned long long vis = 0, bad = 0;
        if (needs_mask) {
          if (valid) {
            const bool page_ok = run.pages_ok || (unsigned)__ldcg(bt + (int)it) < (unsigned)P.n_pages;
            vis = tree_visible(P, sq, token, lo, (run.page0 + (int)(it - it_first)) * TR_KEYS, page_ok, word0);
          }
          const int e = looks % TR_LOOKS;
          TR_WAIT(&S.look_full[ROWS2 ? 0 : h][e], (looks / TR_LOOKS) & 1, 507)
          bad = *(volatile unsigned long long*)&S.bad[ROWS2 ? 0 : h][e];
          looks++;
        }
        if (warp_active) {
          tc_fence_after();
          float sc[TR_KEYS];
          {
            uint32_t (&r)[TR_KEYS] = reinterpret_cast<uint32_t (&)[TR_KEYS]>(sc);
            tmem_ld32(lane_addr + b * TR_KEYS, reinterpret_cast<uint32_t (&)[32]>(r[0]));
            tmem_ld32(lane_addr + b * TR_KEYS + 32, reinterpret_cast<uint32_t (&)[32]>(r[32]));
            tmem_ld_wait();
          }
          if (needs_mask) {
            const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
            for (int e = 0; e < 32; e++) {
              sc[e] = (v0 >> e) & 1 ? sc[e] : -INFINITY;
              sc[32 + e] = (v1 >> e) & 1 ? sc[32 + e] : -INFINITY;
            }
          }
          // (four running maxima: one chain would cost more time than everything else a thread does per tile)
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < TR_KEYS; e += 8)
#pragma unroll
            for (int x = 0; x < 4; x++) mx[x] = tr_max3(mx[x], sc[e + 2 * x], sc[e + 2 * x + 1]);
          const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * to_log2;     // scale > 0
          // the reference moves only when the row's maximum has outgrown it by more than 8 (a factor 256)
          const bool grow = tile_max > m_ref + 8.0f;
          const float corr = grow ? tr_exp2(m_ref - tile_max) : 1.0f;
          if (grow) m_ref = tile_max;
          const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
          uint32_t packed[TR_KEYS / 2];
          const uint64_t mul2 = tr_pair(to_log2, to_log2), neg2 = tr_pair(-m_use, -m_use);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < TR_KEYS; e += 2) {
            float x0, x1;
            tr_split(tr_fma2(tr_pair(sc[e], sc[e + 1]), mul2, neg2), x0, x1);
            // ROWS2: a quarter of them without the exponentials' unit, which eight full warps wait for (64 sequences of 4,000
            // tokens: 4 % less; where rows are few it costs 4 %)
            float p0 = x0, p1 = x1;
            if (ROWS2 && (e & 6) == 6) tr_exp2_pair(p0, p1);
            else { p0 = tr_exp2(x0); p1 = tr_exp2(x1); }
            // P V takes them as bfloat16, off by at most 2^-8 of themselves; the sum runs over the same rounded values, so that
            // a row's weights add up to one and what the values have in common is not touched
            uint32_t u;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(p1), "f"(p0));
            sum2[(e >> 1) & 1] = tr_add2(sum2[(e >> 1) & 1], tr_pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)));
            packed[e >> 1] = u;
          }
          float sum[4], total;
          tr_split(sum2[0], sum[0], sum[1]); tr_split(sum2[1], sum[2], sum[3]);
          const bool move = __any_sync(0xffffffffu, grow);
          if (!first && (move || bad)) {                 // P V of this half's tile before is in O
            const uint32_t before = it - STEP;
            TR_WAIT(&S.pv_full[h][before % STAGES], (before / STAGES) & 1, 508)
          }
          if (!first && move) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t r[32];
              tmem_ld32(o_addr + c, r);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * corr);
              tmem_st32(o_addr + c, r);
            }
          }
          total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
          if (bad) {                                     // what values that are not finite give to the rows that see them
            tc_fence_after();
            tmem_st_wait();
            tree_add_bad<HD>(bad, vis, lane_addr + b * TR_KEYS, o_addr, to_log2, m_use,
                             reinterpret_cast<const bf16*>(P.v_cache) +
                                 ((size_t)((unsigned)__ldcg(bt + (int)it) < (unsigned)P.n_pages ? __ldcg(bt + (int)it) : 0) * P.n_kv + run.kvh) * TR_KEYS * HD, first);
          }
          if (move) any_large = __any_sync(0xffffffffu, fabsf(m_use) >= TR_LARGE);
          if (any_large) total = tree_large_scores(needs_mask ? vis : ~0ull, lane_addr + b * TR_KEYS, to_log2, m_use);
          else tmem_st32(lane_addr + b * TR_KEYS, packed);           // over the scores
          tmem_st_wait();
          l = fmaf(l, corr, total);
        }
        if (first && quarter == 0 && lane == 0) S.o_ready[h] = bad != 0;   // (`bad` is the same in all of them)
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[h][b]);
        i++;
      }
      if (!ok) break;
      // ---- the run is over
      if (it_mine < it_end) {
        const uint32_t last = it - STEP;
        TR_WAIT(&S.pv_full[h][last % STAGES], (last / STAGES) & 1, 508)
      }
      it = it_end;
      const bool whole = run.from_start && run.to_end;
      const int slot = 2 * blockIdx.x + (run.holds_u0 ? 0 : 1);
      bf16* out_row = reinterpret_cast<bf16*>(P.out) + (size_t)token * P.ldo + (size_t)(run.kvh * gs + head) * HD;
      bf16* to[4];                                       // the rows of this lane's group of four
#pragma unroll
      for (int k = 0; k < 4; k++)
        to[k] = reinterpret_cast<bf16*>(__shfl_sync(0xffffffffu, valid ? (unsigned long long)out_row : 0ull, (lane & ~3) + k));
      tc_fence_after();
      if (ROWS2) {
        if (warp_active) {
          const float inv = 1.0f / l;
          float4* po = P.part_o + (size_t)slot * (HD / 4) * 256 + h * 128 + row;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            float o[32];
            tmem_ld32f(o_addr + c, o);                   // (all lanes take part; only valid rows store)
            tmem_ld_wait();
            if (whole) {
              uint4 w[4];
#pragma unroll
              for (int e = 0; e < 4; e++)
                w[e] = make_uint4(tr_pack(l, o[8 * e] * inv, o[8 * e + 1] * inv), tr_pack(l, o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                  tr_pack(l, o[8 * e + 4] * inv, o[8 * e + 5] * inv), tr_pack(l, o[8 * e + 6] * inv, o[8 * e + 7] * inv));
              tr_turn(w);
#pragma unroll
              for (int k = 0; k < 4; k++)
                if (to[k]) *reinterpret_cast<uint4*>(to[k] + c + 8 * (lane & 3)) = w[k];
            } else if (valid) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                po[((c + e) >> 2) * 256] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
          if (valid && !whole) P.part_ml[(size_t)slot * 256 + h * 128 + row] = make_float2(m_ref, l);
        }
        tc_fence_before();
      } else {
        // both halves hold the same rows: half of the dims for each of a row's two threads
        S.ml[h][row] = make_float2(m_ref, l);
        tc_fence_before();
        if (!tr_meet(&S.run_meet, run_phase++, abort_flag)) { if (lane == 0) TR_FAIL(514); ok = false; break; }
        tc_fence_after();
        if (warp_active) {
          const float2 a0 = S.ml[0][row], a1 = S.ml[1][row];
          const float M = fmaxf(a0.x, a1.x), Mu = M == -INFINITY ? 0.f : M;
          const float f0 = tr_exp2(a0.x - Mu), f1 = tr_exp2(a1.x - Mu);
          const float L = f0 * a0.y + f1 * a1.y, inv = 1.0f / L;
          // a half that had no page in this run left its accumulator alone; one that saw no key of the row has nothing to
          // give, whatever lies in it
          const bool has0 = run.n > 1 || (it_first & 1) == 0, has1 = run.n > 1 || (it_first & 1) == 1;
          float4* po = P.part_o + (size_t)slot * (HD / 4) * 128 + row;
#pragma unroll 1
          for (int c = h * (HD / 2); c < (h + 1) * (HD / 2); c += 32) {
            float o[32];
            uint32_t r[32];
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = 0.f;
            if (has0) {
              tmem_ld32(lane_base + COL_PV + c, r);
              tmem_ld_wait();
              if (a0.x != -INFINITY) {
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = f0 * __uint_as_float(r[e]);
              }
            }
            if (has1) {
              tmem_ld32(lane_base + 256 + COL_PV + c, r);
              tmem_ld_wait();
              if (a1.x != -INFINITY) {
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = fmaf(f1, __uint_as_float(r[e]), o[e]);
              }
            }
            if (whole) {
              uint4 w[4];
#pragma unroll
              for (int e = 0; e < 4; e++)
                w[e] = make_uint4(tr_pack(L, o[8 * e] * inv, o[8 * e + 1] * inv), tr_pack(L, o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                  tr_pack(L, o[8 * e + 4] * inv, o[8 * e + 5] * inv), tr_pack(L, o[8 * e + 6] * inv, o[8 * e + 7] * inv));
              tr_turn(w);
#pragma unroll
              for (int k = 0; k < 4; k++)
                if (to[k]) *reinterpret_cast<uint4*>(to[k] + c + 8 * (lane & 3)) = w[k];
            } else if (valid) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                po[((c + e) >> 2) * 128] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
          if (valid && !whole && h == 0) P.part_ml[(size_t)slot * 128 + row] = make_float2(M, L);
        }
        tc_fence_before();
        if (!tr_meet(&S.run_meet, run_phase++, abort_flag)) { if (lane == 0) TR_FAIL(514); ok = false; break; }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.run_empty[r % TR_RUNS]);
    }
  } else {
    // ---------------------------------------------------------------- the walk over the list
    // A run is described here while the ones before it are worked on: what it takes from memory would otherwise stand
    // between two runs of every other warp.  And the values of masked tiles are looked through as they come, ahead of the
    // softmax warps (with these doing it themselves a masked tile took 3 us where the others took 1.2).
    const TreeCursor<false> begin = cur;
    int described = 0, r = 0, t = 0;                       // runs described, the run and the tile of it that is next to be looked at
    uint32_t it0 = 0, looks[2] = {0, 0}, idle = 0;         // tiles in front of that run, masked tiles of the halves
    bool more = true;
    while (more || r < described) {
      bool moved = false;
      if (more && (described < TR_RUNS || __all_sync(0xffffffffu, mbar_test_wait(&S.run_empty[described % TR_RUNS], ((described / TR_RUNS) - 1) & 1)))) {
        TreeRun& run = S.runs[described % TR_RUNS];
        if (lane == 0) cur.next(P, run);
        __syncwarp();
        const int n = run.n;
        if (lane == 0) mbar_arrive(&S.run_full[described % TR_RUNS]);
        if (n == 0) more = false;
        else {
          // what only the softmax warps ask for, while the first keys are fetched: the furthest window edge of the tile's
          // rows (of both halves), whether all pages lie in the pool
          int edge = 0;
          if (P.window > 0) {
            const int per = half_tokens * (ROWS2 ? 2 : 1), t0 = run.s.row0 + run.rt * per, t1 = min(t0 + per, run.s.row0 + run.s.n_new);
            for (int x = t0 + lane; x < t1; x += 32) edge = max(edge, __ldcg(P.token_pos + x) - P.window + 1);
            edge = __reduce_max_sync(0xffffffffu, edge);
          }
          const int* bt = P.block_table + (size_t)run.b * P.bt_stride + run.page0;
          bool ok = true;
#pragma unroll 8
          for (int x = lane; x < n; x += 32) ok &= (unsigned)__ldcg(bt + x) < (unsigned)P.n_pages;
          ok = __all_sync(0xffffffffu, ok);
          if (lane == 0) {
            run.clean0 = min(max((int)(((unsigned)edge + TR_KEYS - 1) / TR_KEYS) - run.page0, 0), n);
            run.clean1 = ok ? min(max(run.s.base / TR_KEYS - run.page0, 0), n) : 0;
            run.pages_ok = ok;
            mbar_arrive(&S.run_seen[described % TR_RUNS]);
          }
          described++;
        }
        __syncwarp();
        moved = true;
      }
      if (r < described) {
        const TreeRun& run = S.runs[r % TR_RUNS];
        if (t >= run.clean0 && t < run.clean1) t = run.clean1;
        if (t >= run.n) {
          it0 += run.n;
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.run_empty[r % TR_RUNS]);
          r++; t = 0;
          moved = true;
        } else {
          // (a barrier tells a phase from the one before it only: it is asked once the tile's values are on their way)
          const uint32_t it = it0 + t;
          const int s = it % STAGES;
          if (__all_sync(0xffffffffu, *(volatile uint32_t*)&S.v_asked > it && mbar_test_wait(&S.v_full[s], (it / STAGES) & 1))) {
            const int h = ROWS2 ? 0 : it & 1, e = (h ? looks[1]++ : looks[0]++) % TR_LOOKS;
            const unsigned long long bad = tree_look_through<HD>(reinterpret_cast<uint4*>(S.v[s]));
            if (lane == 0) {
              *(volatile unsigned long long*)&S.bad[h][e] = bad;
              mbar_arrive(&S.look_full[h][e]);
            }
            __syncwarp();
            t++;
            moved = true;
          }
        }
      }
      if (moved) { idle = 0; continue; }
      __nanosleep(50);
      idle++;
      if (__any_sync(0xffffffffu, idle >= 4u * TC_SPIN_LIMIT || ((idle & 1023u) == 0 && *abort_flag))) { if (lane == 0) TR_FAIL(512); break; }
    }
    if (lane == 0) tree_cut(P, begin, u0, total);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ================================================================ any head size, CUDA cores
// 256 threads take up to 16 R rows of a (sequence, kv head) through pages of 64 keys held in shared memory as float32.  Thread
// (ty, tx) owns rows ty, ty + 16, .. and of them the scores of keys tx, tx + 16, .. and the output dims 4 (tx + 16 j) .. + 3;
// a row's running maximum is kept by its sixteen threads alike, its sum by each for its own keys until the end.  Everything is
// float32; the exponentials are the hardware's, off by 2^-22 of themselves.  What bounds it is multiplications and what shared
// memory delivers to them (12 of every 16 cycles): with rows dealt out one by one every warp has
// the same number of them, and the loops are made for 1 to R rows a thread, so that a tree of 28 rows pays for 32 and not for
// 64.  float32 pages come by cp.async: the next keys while this page's values are summed, the next values while the next
// scores are computed.  Measured: 5 sequences of 300 to 2,500 tokens and 3 to 17 drafted ones, 8 kv heads of 4 queries, head size
// 64: 56 us, of which 5 to the first keys, 7 to 8 a page where two blocks share an SM (the multiplications alone would be 4), four
// or five pages a block.
#define TG_THREADS 256

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// f(rows) with the number as a constant, 1 .. R
template <int N> struct RowsTag { static constexpr int value = N; };
template <int R, typename F>
__device__ __forceinline__ void tg_rows(int used, F f) {
  if (used >= R) f(RowsTag<R>());
  else if constexpr (R > 1) tg_rows<R - 1>(used, f);
}

template <typename T, int NC, int R>
__global__ void __launch_bounds__(TG_THREADS, NC == 1 ? (R == 2 ? 3 : 2) : NC == 2 ? (R == 2 ? 2 : 1) : 1)
attention_tree_simple_kernel(const TreeParams P) {
  extern __shared__ __align__(16) float tg_smem[];
  constexpr int ROWS = 16 * R, PK = TR_KEYS + 4;
  // what concerns the run and its rows lies in shared memory, as the registers are the products'
  __shared__ TreeRun run;
  __shared__ unsigned long long row_vis[ROWS];     // which keys of a masked page a row sees
  __shared__ int row_token[ROWS], row_lo[ROWS], edge;
  const int hd = P.head_dim, hp = (hd + 3) & ~3, pitch = hp + 4;
  float* qs = tg_smem;                             // [ROWS][pitch]
  float* ks = qs + ROWS * pitch;                   // [64][pitch]
  float* vs = ks + TR_KEYS * pitch;                // [64][hp]
  float* ps = vs + TR_KEYS * hp;                   // [ROWS][PK]
  pdl_wait();
  long long u0, total;
  TreeCursor<true> cur = tree_start<true>(P, reinterpret_cast<long long*>(tg_smem), u0, total);
  if (threadIdx.x == TG_THREADS - 1) tree_cut(P, cur, u0, total);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const float scale_log2 = P.scale * 1.4426950408889634f;
  const bool direct = sizeof(T) == 4 && hd == hp && (((uintptr_t)P.k_cache | (uintptr_t)P.v_cache) & 15) == 0;
  const bool q_direct = sizeof(T) == 4 && hd == hp && ((uintptr_t)P.q & 15) == 0 && P.ldq % 4 == 0;
  // a page's keys (or values) into rows of `to` that lie `step` apart; nothing of a page outside the pool
  auto fetch = [&](const void* cache, int pg, int kvh, float* to, int step) {
    if ((unsigned)pg < (unsigned)P.n_pages) {
      const T* from = reinterpret_cast<const T*>(cache) + ((size_t)pg * P.n_kv + kvh) * TR_KEYS * hd;
      if (direct) {
        const int c4 = hp >> 2;
        for (int e = tid; e < TR_KEYS * c4; e += TG_THREADS) cp_async16(to + (e / c4) * step + 4 * (e % c4), reinterpret_cast<const float4*>(from) + e);
      } else {
        for (int e = tid; e < TR_KEYS * hp; e += TG_THREADS) {
          const int r = e / hp, d = e % hp;
          to[r * step + d] = d < hd ? ld_fresh(from + (size_t)r * hd + d) : 0.f;
        }
      }
    }
    cp_async_commit();
  };
  for (;;) {
    __syncthreads();                               // (the run before, or the start, may still be reading)
    if (tid == 0) { cur.next(P, run); edge = 0; }
    __syncthreads();
    if (run.n == 0) break;
    const int r0 = run.rt * run.s.tile_rows, n_rows = min(run.s.n_new * P.gs - r0, run.s.tile_rows);
    const int* bt = P.block_table + (size_t)run.b * P.bt_stride + run.page0;
    int pg = __ldcg(bt);
    fetch(P.k_cache, pg, run.kvh, ks, pitch);
    const int used = (n_rows + 15) >> 4;           // rows of a thread
    for (int r = ty; r < n_rows; r += 16) {        // (a row behind the last one: whatever lies there, and nobody looks at it)
      const T* from = reinterpret_cast<const T*>(P.q) + (size_t)(run.s.row0 + (r0 + r) / P.gs) * P.ldq +
                      (size_t)(run.kvh * P.gs + (r0 + r) % P.gs) * hd;
      if (q_direct) {
        for (int d = 4 * tx; d < hp; d += 64) cp_async16(qs + r * pitch + d, from + d);
      } else {
        for (int d = tx; d < hp; d += 16) qs[r * pitch + d] = d < hd ? ld_fresh(from + d) : 0.f;
      }
    }
    cp_async_commit();
    fetch(P.v_cache, pg, run.kvh, vs, hp);
    if (tid < ROWS) {
      const int token = tid < n_rows ? run.s.row0 + (r0 + tid) / P.gs : -1;
      const int lo = (P.window > 0 && token >= 0) ? max(__ldcg(P.token_pos + token) - P.window + 1, 0) : 0;
      row_token[tid] = token; row_lo[tid] = lo;
      if (lo > 0) atomicMax(&edge, lo);
    }
    float m[R], l[R];
    float4 acc[R][NC];
#pragma unroll
    for (int e = 0; e < R; e++) {
      m[e] = -INFINITY; l[e] = 0.f;
#pragma unroll
      for (int j = 0; j < NC; j++) acc[e][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = 0; i < run.n; i++) {
      const int key0 = (run.page0 + i) * TR_KEYS;
      const bool page_ok = (unsigned)pg < (unsigned)P.n_pages;
      const int pg_next = i + 1 < run.n ? __ldcg(bt + i + 1) : -1;
      cp_async_wait<1>();                          // this page's keys are here (its values may be on their way)
      __syncthreads();
      const bool masked = key0 + TR_KEYS > run.s.base || key0 < edge || !page_ok;
      if (masked && tid < ROWS)
        row_vis[tid] = row_token[tid] >= 0 ? tree_visible(P, run.s, row_token[tid], row_lo[tid], key0, page_ok, __ldcg(P.mask + (size_t)row_token[tid] * P.words)) : 0;
      float s[R][4];
#pragma unroll
      for (int e = 0; e < R; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[e][j] = 0.f;
      if (page_ok) tg_rows<R>(used, [&](auto rows) {
        constexpr int RR = decltype(rows)::value;
        const float* q0 = qs + ty * pitch;
        const float* k0 = ks + tx * pitch;
#pragma unroll 2
        for (int d = 0; d < hp; d += 4) {
          float4 a[RR];
#pragma unroll
          for (int e = 0; e < RR; e++) a[e] = *reinterpret_cast<const float4*>(q0 + 16 * e * pitch + d);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float4 x = *reinterpret_cast<const float4*>(k0 + 16 * j * pitch + d);
#pragma unroll
            for (int e = 0; e < RR; e++) {
              s[e][j] = fmaf(a[e].x, x.x, s[e][j]); s[e][j] = fmaf(a[e].y, x.y, s[e][j]);
              s[e][j] = fmaf(a[e].z, x.z, s[e][j]); s[e][j] = fmaf(a[e].w, x.w, s[e][j]);
            }
          }
        }
      });
      __syncthreads();                             // the keys are read
      if (i + 1 < run.n) fetch(P.k_cache, pg_next, run.kvh, ks, pitch); else cp_async_commit();
#pragma unroll
      for (int e = 0; e < R; e++) {
        if (e >= used) break;
        float mx = -INFINITY;
        const unsigned long long vis = masked ? row_vis[ty + 16 * e] >> tx : ~0ull;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[e][j] = (vis >> (16 * j)) & 1 ? s[e][j] * scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[e][j]);
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float m_new = fmaxf(m[e], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float corr = tr_exp2(m[e] - m_use);
        m[e] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float p = tr_exp2(s[e][j] - m_use);
          sum += p;
          ps[(ty + 16 * e) * PK + tx + 16 * j] = p;
        }
        l[e] = fmaf(l[e], corr, sum);                // (of this thread's keys: the sixteen are added at the end)
#pragma unroll
        for (int j = 0; j < NC; j++) { acc[e][j].x *= corr; acc[e][j].y *= corr; acc[e][j].z *= corr; acc[e][j].w *= corr; }
      }
      cp_async_wait<1>();                          // its values too
      __syncthreads();
      bool odd = false;
      if (masked) {                                // zero times an infinity is not zero: are there any among the values?
        if (page_ok)
          for (int e = tid; e < TR_KEYS * hp; e += TG_THREADS) odd = odd || !isfinite(vs[e]);
        odd = __syncthreads_or(odd);
      }
      const float* p0 = ps + ty * PK;              // (a row's probabilities come from its own warp)
      if (!page_ok) {
      } else if (odd) {                            // then masked keys are left out, one by one
        for (int k = 0; k < TR_KEYS; k++) {
#pragma unroll
          for (int j = 0; j < NC; j++) {
            const int d = 4 * (tx + 16 * j);
            if (d >= hp) continue;
            const float4 x = *reinterpret_cast<const float4*>(vs + k * hp + d);
#pragma unroll
            for (int e = 0; e < R; e++) {
              if (e >= used || !((row_vis[ty + 16 * e] >> k) & 1)) continue;
              const float p = p0[16 * e * PK + k];
              acc[e][j].x = fmaf(p, x.x, acc[e][j].x); acc[e][j].y = fmaf(p, x.y, acc[e][j].y);
              acc[e][j].z = fmaf(p, x.z, acc[e][j].z); acc[e][j].w = fmaf(p, x.w, acc[e][j].w);
            }
          }
        }
      } else tg_rows<R>(used, [&](auto rows) {
        constexpr int RR = decltype(rows)::value;
#pragma unroll 2
        for (int k = 0; k < TR_KEYS; k += 4) {
          float4 p[RR];
#pragma unroll
          for (int e = 0; e < RR; e++) p[e] = *reinterpret_cast<const float4*>(p0 + 16 * e * PK + k);
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
#pragma unroll
            for (int j = 0; j < NC; j++) {
              const int d = 4 * (tx + 16 * j);
              if (NC * 64 != hp && d >= hp) continue;
              const float4 x = *reinterpret_cast<const float4*>(vs + (k + kk) * hp + d);
#pragma unroll
              for (int e = 0; e < RR; e++) {
                const float w = kk == 0 ? p[e].x : kk == 1 ? p[e].y : kk == 2 ? p[e].z : p[e].w;
                acc[e][j].x = fmaf(w, x.x, acc[e][j].x); acc[e][j].y = fmaf(w, x.y, acc[e][j].y);
                acc[e][j].z = fmaf(w, x.z, acc[e][j].z); acc[e][j].w = fmaf(w, x.w, acc[e][j].w);
              }
            }
        }
      });
      __syncthreads();                             // the values are read
      pg = pg_next;
      if (i + 1 < run.n) fetch(P.v_cache, pg, run.kvh, vs, hp); else cp_async_commit();
    }
    const bool whole = run.from_start && run.to_end;
    const int slot = 2 * blockIdx.x + (run.holds_u0 ? 0 : 1);
#pragma unroll
    for (int e = 0; e < R; e++) {
      const int r = ty + 16 * e;
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
      if (r >= n_rows) continue;
      const float inv = 1.0f / l[e];
      T* op = reinterpret_cast<T*>(P.out) + (size_t)row_token[r] * P.ldo + (size_t)(run.kvh * P.gs + (r0 + r) % P.gs) * hd;
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const int d = 4 * (tx + 16 * j);
        const float y[4] = {acc[e][j].x, acc[e][j].y, acc[e][j].z, acc[e][j].w};
        if (whole) {
#pragma unroll
          for (int x = 0; x < 4; x++)
            if (d + x < hd) op[d + x] = from_float<T>(l[e] == 0.f ? 0.f : y[x] * inv);
        } else if (d < hp) {
          *reinterpret_cast<float4*>(ks + r * pitch + d) = acc[e][j];              // (the keys are read, and no more asked for)
        }
      }
      if (!whole && tx == 0) P.part_ml[(size_t)slot * ROWS + r] = make_float2(m[e], l[e]);
    }
    if (!whole) {                                  // a piece, turned in shared memory: a warp writes rows side by side
      __syncthreads();
      float4* po = P.part_o + (size_t)slot * (hp >> 2) * ROWS;
      for (int x = tid; x < (hp >> 2) * ROWS; x += TG_THREADS) {
        const int r = x % ROWS, chunk = x / ROWS;
        if (r < n_rows) po[x] = *reinterpret_cast<const float4*>(ks + r * pitch + 4 * chunk);
      }
    }
  }
  cp_async_wait<0>();
}

// ================================================================ the pieces of what several CTAs saw
// Blocks (c, y) look at the cut between the stretches of CTAs c and c + 1.  The cuts that go through one item share out its
// rows and dims; a lane has a row, so that what a warp reads of a piece lies in one stretch, as the softmax threads, a row each,
// have written it.  A thread has PIECES pieces of 4 CHUNKS dims on their way together, with their maxima and sums: sixteen loads
// whether an item lies in two CTAs or in twenty.
#define TM_WARPS 4
template <typename T, int CHUNKS, int PIECES>
__device__ __forceinline__ void tree_add_up(const TreeParams& P, const TreeCut& cut, int slot_half, int half_rows) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hd = P.head_dim, chunks = (hd + 3) >> 2;               // of four dims
  const int slot_rows = (P.rows_per_tile / half_rows) * slot_half;
  const int wide = (chunks + CHUNKS * TM_WARPS - 1) / (CHUNKS * TM_WARPS), shares = ((cut.n_rows + 31) >> 5) * wide;
  for (int at = blockIdx.y * cut.cuts + (int)blockIdx.x - cut.first; at < shares; at += gridDim.y * cut.cuts) {
    const int r = (at / wide) * 32 + lane, k0 = ((at % wide) * TM_WARPS + warp) * CHUNKS;
    if (r >= cut.n_rows || k0 >= chunks) continue;
    const int srow = (r / half_rows) * slot_half + r % half_rows;
    float M = -INFINITY, L = 0.f;
    float4 acc[CHUNKS];
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = 0; i0 <= cut.cuts; i0 += PIECES) {
      float2 ml[PIECES];
      float4 v[PIECES][CHUNKS];
#pragma unroll
      for (int y = 0; y < PIECES; y++) {
        const bool have = i0 + y <= cut.cuts;
        const size_t slot = 2 * (cut.first + i0 + y) + (i0 + y == 0 ? cut.late : 0);
        ml[y] = have ? __ldcg(P.part_ml + slot * slot_rows + srow) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int j = 0; j < CHUNKS; j++)
          v[y][j] = have && k0 + j < chunks ? __ldcg(P.part_o + (slot * chunks + k0 + j) * slot_rows + srow) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float m = M;
#pragma unroll
      for (int y = 0; y < PIECES; y++) m = fmaxf(m, ml[y].x);
      const float mu = m == -INFINITY ? 0.f : m, corr = exp2f(M - mu);
      M = m;
      L *= corr;
#pragma unroll
      for (int j = 0; j < CHUNKS; j++) { acc[j].x *= corr; acc[j].y *= corr; acc[j].z *= corr; acc[j].w *= corr; }
#pragma unroll
      for (int y = 0; y < PIECES; y++) {
        const float w = exp2f(ml[y].x - mu);
        L = fmaf(w, ml[y].y, L);
        if (w != 0.f) {                            // (no key seen: the piece may hold anything)
#pragma unroll
          for (int j = 0; j < CHUNKS; j++) {
            acc[j].x = fmaf(w, v[y][j].x, acc[j].x); acc[j].y = fmaf(w, v[y][j].y, acc[j].y);
            acc[j].z = fmaf(w, v[y][j].z, acc[j].z); acc[j].w = fmaf(w, v[y][j].w, acc[j].w);
          }
        }
      }
    }
    const int flat = cut.flat0 + r;
    const float inv = 1.0f / L;
    T* op = reinterpret_cast<T*>(P.out) + (size_t)(flat / P.gs) * P.ldo + (size_t)(cut.kvh * P.gs + flat % P.gs) * hd + 4 * k0;
    if (sizeof(T) == 2 && P.out_by_16 && CHUNKS % 2 == 0) {
#pragma unroll
      for (int j = 0; j + 1 < CHUNKS; j += 2)
        if (k0 + j < chunks)
          *reinterpret_cast<uint4*>(op + 4 * j) = make_uint4(tr_pack(L, acc[j].x * inv, acc[j].y * inv), tr_pack(L, acc[j].z * inv, acc[j].w * inv),
                                                             tr_pack(L, acc[j + 1].x * inv, acc[j + 1].y * inv), tr_pack(L, acc[j + 1].z * inv, acc[j + 1].w * inv));
    } else {
#pragma unroll
      for (int j = 0; j < CHUNKS; j++) {
        const float y[4] = {acc[j].x, acc[j].y, acc[j].z, acc[j].w};
#pragma unroll
        for (int d = 0; d < 4; d++)
          if (4 * (k0 + j) + d < hd) op[4 * j + d] = from_float<T>(L == 0.f ? 0.f : y[d] * inv);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * TM_WARPS, 4)
attention_tree_merge_kernel(const TreeParams P, int slot_half, int half_rows) {
  pdl_wait();
  TreeCut cut;                                     // (written by the kernel before, and read past L1)
#pragma unroll
  for (int x = 0; x < 2; x++) reinterpret_cast<int4*>(&cut)[x] = __ldcg(reinterpret_cast<const int4*>(P.cut + blockIdx.x + 1) + x);
  if (cut.cuts == 0) return;
  if (cut.cuts == 1) tree_add_up<T, 8, 2>(P, cut, slot_half, half_rows);
  else if (cut.cuts < 4) tree_add_up<T, 4, 4>(P, cut, slot_half, half_rows);
  else tree_add_up<T, 1, 16>(P, cut, slot_half, half_rows);
}

// ---------------------------------------------------------------- host side
static int tree_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                    const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return STRATUM_ERR_LIMIT;
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : STRATUM_ERR_SHAPE;
}

// (The opt-in to more shared memory is the current device's, and a cheap call: it is made at every launch.)
template <int HD, bool ROWS2>
static int launch_tree_tc(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TreeParams& P, int G,
                          cudaStream_t stream) {
  const size_t smem = sizeof(TreeSmem<HD, ROWS2>);
  auto kern = attention_tree_tc_kernel<HD, ROWS2>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  return launch_pdl(kern, dim3(G), dim3(TR_THREADS), smem, stream, mq, mk, mv, P);
}

static size_t simple_smem(int head_dim, int rows, int n_seqs) {
  const int hp = (head_dim + 3) & ~3;
  const size_t tiles = ((size_t)(rows + TR_KEYS) * (hp + 4) + (size_t)TR_KEYS * hp + (size_t)rows * (TR_KEYS + 4)) * sizeof(float);
  const size_t sums = (size_t)(n_seqs + 1) * sizeof(long long);
  return tiles > sums ? tiles : sums;
}

template <typename T, int NC, int R>
static int launch_tree_simple(const TreeParams& P, int G, cudaStream_t stream) {
  const size_t smem = simple_smem(P.head_dim, 16 * R, P.n_seqs);
  auto kern = attention_tree_simple_kernel<T, NC, R>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
  if (e != cudaSuccess) return (int)e;
  return launch_pdl(kern, dim3(G), dim3(TG_THREADS), smem, stream, P);
}
template <typename T>
static int launch_tree_simple_of(const TreeParams& P, int G, cudaStream_t stream) {
  if (P.rows_per_tile == 32)
    return P.head_dim <= 64 ? launch_tree_simple<T, 1, 2>(P, G, stream)
         : P.head_dim <= 128 ? launch_tree_simple<T, 2, 2>(P, G, stream) : launch_tree_simple<T, 4, 2>(P, G, stream);
  return P.head_dim <= 64 ? launch_tree_simple<T, 1, 4>(P, G, stream)
       : P.head_dim <= 128 ? launch_tree_simple<T, 2, 4>(P, G, stream) : launch_tree_simple<T, 4, 4>(P, G, stream);
}

// Slot rows of a launch's scratch: tensor: the tcgen05 kernel, of 128 rows a half; else the CUDA-core kernel, of 32 or 64
// rows.  many: a tree has more rows than the smaller one of the two holds.
STRATUM_EXPORT int stratum_attention_tree_slot_rows(int tensor, int many) { return tensor ? (many ? 256 : 128) : (many ? 64 : 32); }

// CTAs of a launch (the scratch has two slots of rows for each): one per SM, or of the CUDA-core kernel as many as find room.
STRATUM_EXPORT int stratum_attention_tree_ctas(int tensor, int many, int head_dim) {
  if (tensor) return sm_count();
  const int most = head_dim <= 64 ? (many ? 2 : 3) : head_dim <= 128 ? (many ? 1 : 2) : 1;     // (by registers: see the kernel)
  const int room = (int)((size_t)(227 * 1024) / (simple_smem(head_dim, many ? 64 : 32, 0) + 3 * 1024));
  return sm_count() * (room < 1 ? 1 : room < most ? room : most);
}

// Scratch: part_o float32 [G][2][head_dim rounded up to 4, / 4][slot rows][4], part_ml float32 [G][2][slot rows][2], cut 32 bytes
// a CTA.
// One call's numbers, as the launcher packs them (pointers first, then 8 bytes, then 4).
struct TreeCall {
  const void *q, *k_cache, *v_cache, *token_pos, *mask, *seq_start, *seq_len, *block_table;
  void *out, *part_o, *part_ml, *cut, *status;
  long long n_pages;
  int dtype, ldq, ldo, words, bt_stride, bt_width, n_tokens, n_seqs, n_q, n_kv, head_dim, page_tokens, window, tensor, many;
  float scale;
};

STRATUM_EXPORT int stratum_attention_tree(const TreeCall* call, cudaStream_t stream) {
  const TreeCall& a = *call;
  const int n_tokens = a.n_tokens, n_seqs = a.n_seqs, n_q = a.n_q, n_kv = a.n_kv, head_dim = a.head_dim, dtype = a.dtype;
  const int ldq = a.ldq, ldo = a.ldo, tensor = a.tensor, many = a.many;
  const long long n_pages = a.n_pages;
  if (n_tokens <= 0 || n_seqs <= 0) return 0;
  if (dtype != STRATUM_DT_F32 && dtype != STRATUM_DT_BF16) return STRATUM_ERR_DTYPE;
  if (n_kv < 1 || n_q < 1 || n_q % n_kv != 0 || a.page_tokens != TR_KEYS || head_dim < 1 || head_dim > 256) return STRATUM_ERR_SHAPE;
  if (a.words < 1 || a.bt_width < 1 || a.window < 0 || n_pages < 1) return STRATUM_ERR_SHAPE;
  if (n_seqs > TR_MAX_SEQS || n_pages * n_kv * TR_KEYS > 0x7fffffffLL) return STRATUM_ERR_LIMIT;
  const int gs = n_q / n_kv;
  if ((long long)n_tokens * gs > 0x7fffffffLL) return STRATUM_ERR_LIMIT;
  if (!a.part_o || !a.part_ml || !a.cut || !a.status) return STRATUM_ERR_ALIGN;
  TreeParams P;
  P.token_pos = (const int*)a.token_pos; P.mask = (const unsigned long long*)a.mask; P.words = a.words;
  P.seq_start = (const int*)a.seq_start; P.seq_len = (const int*)a.seq_len;
  P.block_table = (const int*)a.block_table; P.bt_stride = a.bt_stride; P.bt_width = a.bt_width;
  P.q = a.q; P.ldq = ldq; P.k_cache = a.k_cache; P.v_cache = a.v_cache; P.out = a.out; P.ldo = ldo;
  P.part_o = (float4*)a.part_o; P.part_ml = (float2*)a.part_ml; P.cut = (TreeCut*)a.cut; P.status = (int*)a.status;
  P.n_tokens = n_tokens; P.n_seqs = n_seqs; P.n_q = n_q; P.n_kv = n_kv; P.gs = gs; P.head_dim = head_dim;
  P.item_units = tensor ? 7 : 8;                 // (see the list of units)
  P.out_by_16 = head_dim % 8 == 0 && ldo % 8 == 0 && ((uintptr_t)a.out & 15) == 0;
  P.window = a.window; P.n_pages = (int)n_pages; P.scale = a.scale;
  const int G = stratum_attention_tree_ctas(tensor, many, head_dim);
  int st, slot_half, half_rows;
  if (tensor) {
    if (dtype != STRATUM_DT_BF16 || (head_dim != 64 && head_dim != 128) || gs > 128 || !(a.scale > 0.f)) return STRATUM_ERR_SHAPE;
    if (ldq % 8 != 0 || ldo % 8 != 0) return STRATUM_ERR_ALIGN;
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.out) & 15) return STRATUM_ERR_ALIGN;
    const int half_tokens = 128 / gs;
    slot_half = 128; half_rows = half_tokens * gs;
    P.rows_per_tile = half_rows * (many ? 2 : 1);
    CUtensorMap mq, mk, mv;
    {  // q as [tokens][n_q heads][head_dim]; a box is 64 dims x gs heads x half_tokens tokens: rows token * gs + head
      cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)n_q, (cuuint64_t)n_tokens};
      cuuint64_t strides[2] = {(cuuint64_t)head_dim * sizeof(bf16), (cuuint64_t)ldq * sizeof(bf16)};
      cuuint32_t box[3] = {64, (cuuint32_t)gs, (cuuint32_t)half_tokens};
      if ((st = tree_map(&mq, a.q, 3, dims, strides, box)) != 0) return st;
    }
    {  // the cache as [pages * n_kv * 64 rows][head_dim]; a box is 64 dims x 64 keys
      cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)n_pages * n_kv * TR_KEYS};
      cuuint64_t strides[1] = {(cuuint64_t)head_dim * sizeof(bf16)};
      cuuint32_t box[2] = {64, TR_KEYS};
      if ((st = tree_map(&mk, a.k_cache, 2, dims, strides, box)) != 0) return st;
      if ((st = tree_map(&mv, a.v_cache, 2, dims, strides, box)) != 0) return st;
    }
    if (head_dim == 64) st = many ? launch_tree_tc<64, true>(mq, mk, mv, P, G, stream) : launch_tree_tc<64, false>(mq, mk, mv, P, G, stream);
    else st = many ? launch_tree_tc<128, true>(mq, mk, mv, P, G, stream) : launch_tree_tc<128, false>(mq, mk, mv, P, G, stream);
  } else {
    slot_half = half_rows = P.rows_per_tile = many ? 64 : 32;
    st = dtype == STRATUM_DT_F32 ? launch_tree_simple_of<float>(P, G, stream) : launch_tree_simple_of<bf16>(P, G, stream);
  }
  if (st != 0 || G < 2) return st;
  const dim3 grid(G - 1, 4), block(32 * TM_WARPS);               // (one wave: four blocks to an SM)
  if (dtype == STRATUM_DT_F32) return launch_pdl(attention_tree_merge_kernel<float>, grid, block, 0, stream, P, slot_half, half_rows);
  return launch_pdl(attention_tree_merge_kernel<bf16>, grid, block, 0, stream, P, slot_half, half_rows);
}
