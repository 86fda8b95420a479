// What a paged cache does besides growing: whole pages are copied (a sequence begins as a copy of another one), and the
// rows of the drafted tokens that were kept move together behind the tokens in front of them.  Both work on a group's keys
// and values in all its layers in one launch, and move bytes: any element type.
//
// A page of a layer is one stretch of n_kv * 64 * head_dim elements, a token's row of a (page, head) one of head_dim.
#include "common.cuh"

static int sms() {                                  // of the current device
  int n = 0, dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

// ================================================================ pages
// The pairs travel with the launch.  Pages are cut into pieces of eight rounds of a block; a block takes every (grid)th piece, each
// thread 16 bytes (or 4, or 1, where the sizes ask for that) at a time, eight on their way together.  Bound by memory: 97
// pairs in 16 layers of 8 heads of 128 (814 MB read and written) in 131 us, 6.2 TB/s, 0.95 of a plain copy.
#define CM_PAIRS 480
#define CM_THREADS 256
struct PagePairs { int src[CM_PAIRS], dst[CM_PAIRS]; };

template <typename V>
__global__ void __launch_bounds__(CM_THREADS)
copy_pages_kernel(uint8_t* a, uint8_t* b, long long pages, long long bytes_a, long long bytes_b, int layers, int n_pairs,
                  const __grid_constant__ PagePairs pairs) {
  pdl_wait();
  constexpr int UNROLL = 8, PIECE = CM_THREADS * UNROLL;           // in units of V
  const long long va = bytes_a / sizeof(V), vb = bytes_b / sizeof(V);
  const long long pa = (va + PIECE - 1) / PIECE, pb = (vb + PIECE - 1) / PIECE, per_page = pa + pb;
  const long long total = per_page * layers * n_pairs;
  for (long long w = blockIdx.x; w < total; w += gridDim.x) {
    const long long page = w / per_page;
    const int layer = (int)(page / n_pairs), pair = (int)(page % n_pairs);
    long long piece = w % per_page;
    const bool second = piece >= pa;
    if (second) piece -= pa;
    const long long n = second ? vb : va;
    V* base = reinterpret_cast<V*>(second ? b : a) + layer * pages * n;
    const V* from = base + pairs.src[pair] * n;
    V* to = base + pairs.dst[pair] * n;
    const long long i0 = piece * PIECE + threadIdx.x;
    V x[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; j++) if (i0 + j * CM_THREADS < n) x[j] = __ldcg(from + i0 + j * CM_THREADS);
#pragma unroll
    for (int j = 0; j < UNROLL; j++) if (i0 + j * CM_THREADS < n) to[i0 + j * CM_THREADS] = x[j];
  }
}

// a, b: [layers][pages][bytes_a | bytes_b], b may be null (bytes_b 0).  Pages src[i] -> dst[i]; no page is written that
// another pair reads or writes (the caller has looked).
STRATUM_EXPORT int stratum_copy_pages(void* a, void* b, long long pages, long long bytes_a, long long bytes_b, int layers,
                                      const int* src, const int* dst, int n_pairs, cudaStream_t stream) {
  if (n_pairs <= 0 || layers <= 0) return 0;
  if (n_pairs > CM_PAIRS) return STRATUM_ERR_LIMIT;
  if (!a || bytes_a <= 0 || bytes_b < 0 || (bytes_b > 0 && !b)) return STRATUM_ERR_SHAPE;
  PagePairs pairs;
  for (int i = 0; i < n_pairs; i++) {
    if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages) return STRATUM_ERR_LIMIT;
    pairs.src[i] = src[i]; pairs.dst[i] = dst[i];
  }
  for (int i = n_pairs; i < CM_PAIRS; i++) pairs.src[i] = pairs.dst[i] = 0;
  const unsigned long long all = (unsigned long long)(uintptr_t)a | (uintptr_t)b | (unsigned long long)bytes_a | (unsigned long long)bytes_b;
  const int unit = (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : 1;
  const long long piece = (long long)unit * CM_THREADS * 8;
  const long long total = ((bytes_a + piece - 1) / piece + (bytes_b + piece - 1) / piece) * layers * n_pairs;
  const long long most = (long long)sms() * 8;
  const dim3 grid((unsigned)(total < most ? total : most));
  uint8_t* pa = (uint8_t*)a;
  uint8_t* pb = (uint8_t*)b;
  if (unit == 16) return launch_pdl(copy_pages_kernel<uint4>, grid, dim3(CM_THREADS), 0, stream, pa, pb, pages, bytes_a, bytes_b, layers, n_pairs, pairs);
  if (unit == 4) return launch_pdl(copy_pages_kernel<uint32_t>, grid, dim3(CM_THREADS), 0, stream, pa, pb, pages, bytes_a, bytes_b, layers, n_pairs, pairs);
  return launch_pdl(copy_pages_kernel<uint8_t>, grid, dim3(CM_THREADS), 0, stream, pa, pb, pages, bytes_a, bytes_b, layers, n_pairs, pairs);
}

// ================================================================ kept rows
// Sequence s has seq_len[s] keys of which the last n = seq_start[s + 1] - seq_start[s] are drafted ones; path[seq_start[s] + j],
// j = 1 .. kept[s], says which of them is kept in the j-th place.  Row base + path[j] of every layer, head, keys and values
// goes to base + j.  The path rises and path[j] >= j (nodes stand behind their parents), so rows move towards the front
// only and, taken in ascending stretches of which each is read before it is written, none is written that is still to be read.
//
// A warp owns a (sequence, layer, head, keys or values) and moves its rows CR_ROWS at a time; what it moves is its own, so
// nothing waits for other warps.  Measured: 32 sequences that keep up to 15 of 31 drafted rows, 32 layers of 8 heads of 128 (77 MB)
// in 20 us, 3.8 TB/s: a warp's few rows are one chain (what the path says, where it lies, the rows), which 16,384 warps hide
// only in part.
#define CR_THREADS 256
#define CR_ROWS 8

// One call's numbers, as the launcher packs them.  k: [layers][pages][heads_k][page_tokens][bytes_k], v likewise (null:
// heads_v 0).
struct KeepRows {
  uint8_t *k, *v;
  const int *block_table, *seq_start, *seq_len, *path, *kept;
  long long pages;
  int heads_k, heads_v, bytes_k, bytes_v, layers, page_tokens, bt_stride, bt_width, n_tokens, n_seqs;
};

template <typename V>
__global__ void __launch_bounds__(CR_THREADS, 4)
keep_rows_kernel(const KeepRows P, int per_seq) {
  __shared__ V* from_s[CR_THREADS / 32][32];
  __shared__ V* to_s[CR_THREADS / 32][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = blockIdx.x / per_seq;
  int w = (blockIdx.x % per_seq) * (CR_THREADS / 32) + warp;       // layer, then keys' heads and values' heads
  if (w >= P.layers * (P.heads_k + P.heads_v)) return;
  // (fetched together: what the path says, where it lies and how much of it holds)
  const int a0 = __ldcg(P.seq_start + s), a1 = __ldcg(P.seq_start + s + 1), len = __ldcg(P.seq_len + s), kept = __ldcg(P.kept + s);
  const int layer = w / (P.heads_k + P.heads_v);
  w %= P.heads_k + P.heads_v;
  const bool second = w >= P.heads_k;
  const int head = second ? w - P.heads_k : w, heads = second ? P.heads_v : P.heads_k;
  const int units = (second ? P.bytes_v : P.bytes_k) / (int)sizeof(V);              // of a row
  const int a = min(max(a0, 0), P.n_tokens), n = min(max(a1, a), P.n_tokens) - a;
  const int base = len - n, last = min(kept, n - 1);
  if (last < 1 || base < 0) return;
  V* all = reinterpret_cast<V*>(second ? P.v : P.k) + (long long)layer * P.pages * heads * P.page_tokens * units;
  const int* bt = P.block_table + (long long)s * P.bt_stride;
  // where position p of this head lies, or null
  auto at = [&](int p) -> V* {
    const int i = p / P.page_tokens;
    if (i >= P.bt_width) return nullptr;
    const int pg = __ldcg(bt + i);
    if (pg < 0 || pg >= P.pages) return nullptr;
    return all + (((long long)pg * heads + head) * P.page_tokens + p % P.page_tokens) * units;
  };
  // a row takes `g` lanes (the next power of two of its units, a warp at most); 32 / g rows go side by side
  const int g = units >= 32 ? 32 : units <= 1 ? 1 : 1 << (32 - __clz(units - 1)), side = 32 / g, sub = lane / g, unit = lane % g;
  int before = 0;                                  // the path's entry in front; one that does not rise ends it
  for (int j0 = 1; j0 <= last; j0 += 32) {
    const int j = j0 + lane;
    const int node = j <= last ? __ldcg(P.path + a + j) : -1;
    int prev = __shfl_up_sync(0xffffffffu, node, 1);
    if (lane == 0) prev = before;
    const unsigned wrong = __ballot_sync(0xffffffffu, j > last || node <= prev || node >= n);
    const int count = wrong ? __ffs(wrong) - 1 : 32;
    before = __shfl_sync(0xffffffffu, node, 31);
    V* from = nullptr;
    V* to = nullptr;
    if (lane < count && node != j) { from = at(base + node); to = at(base + j); }
    const bool moves = from && to;
    const unsigned which = __ballot_sync(0xffffffffu, moves);
    const int m = __popc(which), mine = __popc(which & ((1u << lane) - 1));
    __syncwarp();
    if (moves) { from_s[warp][mine] = from; to_s[warp][mine] = to; }
    __syncwarp();
    for (int r0 = 0; r0 < m; r0 += CR_ROWS * side) {              // rows in the path's order: read, then written
      for (int i0 = 0; i0 < units; i0 += g) {
        V x[CR_ROWS];
#pragma unroll
        for (int r = 0; r < CR_ROWS; r++) {
          const int at_ = r0 + r * side + sub;
          if (at_ < m && i0 + unit < units) x[r] = __ldcg(from_s[warp][at_] + i0 + unit);
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < CR_ROWS; r++) {
          const int at_ = r0 + r * side + sub;
          if (at_ < m && i0 + unit < units) to_s[warp][at_][i0 + unit] = x[r];
        }
        __syncwarp();
      }
    }
    if (count < 32) return;
  }
}

STRATUM_EXPORT int stratum_keep_rows(const KeepRows* call, cudaStream_t stream) {
  const KeepRows P = *call;
  if (P.n_seqs <= 0 || P.layers <= 0 || P.n_tokens <= 0) return 0;
  if (!P.k || P.heads_k < 1 || P.bytes_k < 1 || P.heads_v < 0 || (P.heads_v > 0 && (!P.v || P.bytes_v < 1)) || P.page_tokens < 1 ||
      P.bt_width < 1)
    return STRATUM_ERR_SHAPE;
  const long long warps = (long long)P.layers * (P.heads_k + P.heads_v), per_seq = (warps + CR_THREADS / 32 - 1) / (CR_THREADS / 32);
  if (warps > 0x7fffffffLL || per_seq * P.n_seqs > 0x7fffffffLL) return STRATUM_ERR_LIMIT;
  const unsigned long long all = (unsigned long long)(uintptr_t)P.k | (uintptr_t)P.v | (unsigned)P.bytes_k | (unsigned)P.bytes_v;
  const dim3 grid((unsigned)(per_seq * P.n_seqs)), block(CR_THREADS);
  if ((all & 15) == 0) return launch_pdl(keep_rows_kernel<uint4>, grid, block, 0, stream, P, (int)per_seq);
  if ((all & 3) == 0) return launch_pdl(keep_rows_kernel<uint32_t>, grid, block, 0, stream, P, (int)per_seq);
  return launch_pdl(keep_rows_kernel<uint8_t>, grid, block, 0, stream, P, (int)per_seq);
}
