// Drafted tokens against the target: the target's probabilities, and the walk through a sequence's tree of drafts.
//
// Probabilities: p_i = exp((l_i - max) / T) / sum per row of logits; T <= 0 (or no number): one at the largest logit, the
// lowest index among equals.  A logit that is no number counts as -inf; infinite ones share the row evenly; a row without
// any logit above -inf is all zeros.
//
// Verification.  A sequence's nodes are rows seq_start[s] .. seq_start[s + 1] - 1; the first is the token it went on with,
// the others are drafts, each behind its parent.  The walk begins at the first node with d = the target's probabilities
// behind it and mass = 1, and tries the node's children in order, child x with its own number u:
//   drawn from a draft distribution q (that of the parent's row):  taken if u mass q(x) < d(x);  else  d = max(d - mass q, 0)
//     and mass = sum d, unless nothing would be left (after several rejections d = max(p - cover q, 0) with the sum of the
//     masses so far for `cover`, since max(max(a, 0) - b, 0) = max(a - b, 0));
//   looked up, without a distribution:  taken if u mass < d(x);  else  mass = max(mass - d(x), 0) and d(x) = 0, unless nothing
//     would be left: a row of rounded probabilities adds up to a little less than one, so that children that hold all of it
//     may all be refused.  The last one with any weight is then what there is to draw.
// A child that is taken is the next node.  Where none is, the next token is drawn from d: the first index whose running sum
// is over u_0 sum(d), u_0 being the first node's number (the last index with any weight if rounding leaves none).  Whoever
// drafts, the kept tokens and the one behind them are distributed as the target's own draws
// (each rejection leaves the target's distribution less what the draft could have covered, at the scale `mass`).
//
// Probabilities are clamped to [0, 1] on reading (no number: 0).  Everything behind that is in 64 bits: the draw lies between
// two of 10^5 running sums, and with 32 bits one draw in some hundreds would land on the other side of its border.
//
// Both kernels give a row to a cluster of thread blocks, which meet through distributed shared memory.
#include <cooperative_groups.h>
#include <math.h>

#include <atomic>

#include "tc_common.cuh"

namespace cg = cooperative_groups;

// Clusters of C blocks of a kernel that are resident at a time (at most 16 blocks; 0: none).
static int resident_clusters(const void* kernel, int C, int threads) {
  if (C > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) { cudaGetLastError(); return 0; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(threads);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); return 0; }
  return n;
}

// rows clusters of `cluster` blocks each
template <auto kernel, typename... Args>
static int launch_clusters(unsigned rows, unsigned cluster, unsigned threads, cudaStream_t stream, Args... args) {
  if (cluster > 8) {                               // clusters of sixteen: the current device's opt-in
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * cluster);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A block may write to another one's shared memory once that one has begun: everybody says so at the start and looks, when it
// comes to that, whether the others have.
__device__ __forceinline__ void cluster_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_all_begun() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// ================================================================ probabilities
// A row is read once and written once: its values stay in registers, 32 to a thread of a block, the rest of the row in the
// other blocks of the cluster.  A block takes its exponentials against its own largest value, so the blocks meet
// once: each tells the others that value (and where it is) and its sum, and its weights then need one factor.  (A row longer
// than sixteen blocks hold is read a second and a third time.)
//
// With ordinary numbers a weight is a difference, a product and an exponential; infinities, and temperatures that are so large
// or small that the product is none, are told apart once for a block: decided for every value they were fifty instructions
// a value, and the time was theirs (287 us against 224 for 1,024 rows of 128,256, then).
//
// Measured: 1,024 rows of 128,256 in 203 to 210 us from card to card, 5.0 to 5.2 TB/s read and written, 0.77 to 0.79 of a plain copy;
// what is missing is a row's blocks waiting for one another between reading and writing, while the other three or so on their SM
// read or write.  (Where this form took 200: with a meeting of the cluster, whose fence waits for all that a block has under way,
// 225; blocks that stay and take row after row 316; three blocks to an SM, without spills, 226; blocks of 512 threads 203.)
// Nine rows: 5 us, launch and three trips to memory.
#define PR_HELD 32

struct alignas(16) Part { float v, sum; int i, unused; };   // the largest value, the sum of weights against it, where it is first

// 16 bytes to block `rank` of the cluster, whose barrier counts them: nobody waits for a fence, and a block goes on once it has
// heard from all.
__device__ __forceinline__ void tell(const Part* place, const uint64_t* bar, int rank, float v, float sum, int i) {
  asm volatile(
      "{\n\t.reg .b32 a, b;\n\t"
      "mapa.shared::cluster.u32 a, %0, %2;\n\t"
      "mapa.shared::cluster.u32 b, %1, %2;\n\t"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [a], {%3, %4, %5, %6}, [b];\n\t}"
      ::"r"(smem_u32(place)), "r"(smem_u32(bar)), "r"(rank), "r"(__float_as_uint(v)), "r"(__float_as_uint(sum)), "r"(i), "r"(0) : "memory");
}

// A weight against `m`, no less than v and above -inf, in all cases: 1 at the maximum (infinite ones too), 0 at -inf and beside an
// infinite one (there the product may be none: fmaxf drops it).  Halves, as the difference of two numbers may be none of its
// own: with T that large as well the weight is not 0.
__device__ __forceinline__ float any_weight(float v, float m, float to_log2) {
  return v == m ? 1.f : exp2f(2.f * fmaxf((0.5f * v - 0.5f * m) * to_log2, -1000.f));
}
__device__ __forceinline__ float clean(float v) { return fmaxf(v, -INFINITY); }        // (fmaxf drops what is no number)

// W: values of a load and a store (4 where every row begins on 16 bytes)
template <bool HELD, int W, int PR_THREADS>
__global__ void __launch_bounds__(PR_THREADS, 1024 / PR_THREADS)
token_probs_kernel(const float* logits, long long ld, const float* temperature, float* out, long long ldo, int vocab, int slice, int* status) {
  __shared__ float warp_v[PR_THREADS / 32], warp_sum_[PR_THREADS / 32];
  __shared__ int first;
  __shared__ Part told[16];
  __shared__ uint64_t all_told;
  __shared__ int given_up;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    given_up = 0;
    mbar_init(&all_told, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    mbar_expect_tx(&all_told, C * sizeof(Part));
  }
  cluster_begun();
  pdl_wait();
  const int i0 = min(c * slice, vocab), n = min(vocab - i0, slice);
  const float* in = logits + row * ld + i0;
  float* to = out + row * ldo + i0;
  const float t = ld_fresh(temperature + row);
  float x[PR_HELD], v = -INFINITY;
  auto place = [&](int k) { return ((k / W) * PR_THREADS + tid) * W + k % W; };      // of a thread's k-th value in the slice
  if (HELD) {
#pragma unroll
    for (int k = 0; k < PR_HELD; k += W) {
      const int i = place(k);
      if (W == 4 && i + 3 < n) {
        const float4 y = ld_fresh(reinterpret_cast<const float4*>(in + i));
        x[k] = y.x; x[k + W / 4] = y.y; x[k + W / 2] = y.z; x[k + W - 1] = y.w;
      } else {
#pragma unroll
        for (int e = 0; e < W; e++) x[k + e] = i + e < n ? ld_fresh(in + i + e) : -INFINITY;
      }
    }
    if (tid == 0) first = 0x7fffffff;
    float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) { x[k] = clean(x[k]); most[k & 3] = fmaxf(most[k & 3], x[k]); }
    v = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  } else {
    if (tid == 0) first = 0x7fffffff;
    for (int i = tid; i < n; i += PR_THREADS) v = fmaxf(v, ld_fresh(in + i));
  }
  v = warp_max(v);
  if (lane == 0) warp_v[warp] = v;
  __syncthreads();
  const float m = warp_max(warp_v[lane % (PR_THREADS / 32)]);                        // the block's largest value
  const bool greedy = !(t > 0.f);
  const float to_log2 = greedy ? 0.f : 1.4426950408889634f / t;
  // (below 1e-30 a difference that has overflowed may still have a weight)
  const bool ordinary = fabsf(m) < INFINITY && to_log2 > 1e-30f && to_log2 < INFINITY;
  float sum = 0.f;
  if (greedy) {
    if (HELD) {
#pragma unroll
      for (int k = 0; k < PR_HELD; k++) if (x[k] == m && place(k) < n) atomicMin(&first, i0 + place(k));
    } else {
      for (int i = tid; i < n; i += PR_THREADS) if (clean(ld_fresh(in + i)) == m) atomicMin(&first, i0 + i);
    }
  } else if (HELD && ordinary) {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) {
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x[k]) : "f"((x[k] - m) * to_log2));
      part[k & 3] += x[k];
    }
    sum = (part[0] + part[1]) + (part[2] + part[3]);
  } else if (m != -INFINITY) {
    if (HELD) {
#pragma unroll
      for (int k = 0; k < PR_HELD; k++) { x[k] = any_weight(x[k], m, to_log2); sum += x[k]; }
    } else {
      for (int i = tid; i < n; i += PR_THREADS) sum += any_weight(clean(ld_fresh(in + i)), m, to_log2);
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) warp_sum_[warp] = sum;
  __syncthreads();
  cluster_all_begun();
  if (warp == 0) {
    sum = warp_sum(lane < PR_THREADS / 32 ? warp_sum_[lane] : 0.f);
    if (lane < C) tell(&told[c], &all_told, lane, m, sum, first);
  }
  if (!mbar_wait(&all_told, 0, &given_up)) {       // (the others have told this block: none writes here any more)
    atomicCAS(status, 0, 521);
    return;
  }
  const Part p = lane < C ? told[lane] : Part{-INFINITY, 0.f, 0x7fffffff, 0};
  const float M = warp_max(p.v);                   // of the row
  if (greedy || M == -INFINITY) {                  // (the same in the whole cluster)
    const int best = __reduce_min_sync(0xffffffffu, p.v == M ? p.i : 0x7fffffff);    // (-inf: nowhere)
    for (int i = tid; i < n; i += PR_THREADS) to[i] = M != -INFINITY && i0 + i == best ? 1.f : 0.f;
    return;
  }
  const float inv = 1.0f / warp_sum(p.v == -INFINITY ? 0.f : p.sum * any_weight(p.v, M, to_log2));
  const float f = m == -INFINITY ? 0.f : any_weight(m, M, to_log2) * inv;
  if (HELD) {
    if (m == -INFINITY) {
#pragma unroll
      for (int k = 0; k < PR_HELD; k++) x[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < PR_HELD; k += W) {
      const int i = place(k);
      if (W == 4 && i + 3 < n) {
        *reinterpret_cast<float4*>(to + i) = make_float4(x[k] * f, x[k + W / 4] * f, x[k + W / 2] * f, x[k + W - 1] * f);
      } else {
#pragma unroll
        for (int e = 0; e < W; e++) if (i + e < n) to[i + e] = x[k + e] * f;
      }
    }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) to[i] = any_weight(clean(ld_fresh(in + i)), M, to_log2) * inv;
  }
}

// logits float32 [rows][ld], temperature float32 [rows], out float32 [rows][ldo]; out may be logits (the same rows at the same
// distance).  As the launcher packs them.
struct ProbsCall {
  const float *logits, *temperature;
  float* out;
  int* status;
  long long ld, ldo;
  int rows, vocab;
};

STRATUM_EXPORT int stratum_token_probs(const ProbsCall* call, cudaStream_t stream) {
  const float *logits = call->logits, *temperature = call->temperature;
  float* out = call->out;
  int* status = call->status;
  const long long ld = call->ld, ldo = call->ldo;
  const int rows = call->rows, vocab = call->vocab;
  if (rows <= 0 || vocab <= 0) return 0;
  if (rows > (1 << 26) || vocab > (1 << 30)) return STRATUM_ERR_LIMIT;
  const bool four = (((uintptr_t)logits | (uintptr_t)out) & 15) == 0 && (rows == 1 || (ld % 4 == 0 && ldo % 4 == 0));
  const int threads = vocab <= 16 * 256 * PR_HELD ? 256 : 512;
  // enough blocks to hold a row; beyond that, where a few rows leave the GPU empty, blocks of shorter slices
  int C = 1;
  while (C < 16 && ((long long)C * threads * PR_HELD < vocab || (C * 4096 < vocab && (long long)rows * C * 2 <= sm_count()))) C *= 2;
  const int slice = (((vocab + C - 1) / C) + 3) & ~3;
#define PROBS(HELD, W, THREADS) \
  launch_clusters<token_probs_kernel<HELD, W, THREADS>>(rows, C, THREADS, stream, logits, ld, temperature, out, ldo, vocab, slice, status)
  if (slice > threads * PR_HELD) return PROBS(false, 1, 512);
  if (threads == 256) return four ? PROBS(true, 4, 256) : PROBS(true, 1, 256);
  return four ? PROBS(true, 4, 512) : PROBS(true, 1, 512);
#undef PROBS
}

// ================================================================ verification
#define VD_THREADS 512
#define VD_WARPS (VD_THREADS / 32)
#define VD_NODES 1024            // nodes of a sequence that are looked at

struct VerifyParams {
  const float* target;
  const float* draft;                      // null: looked up
  const int* tokens; const int* parents; const int* seq_start; const float* uniform;
  int* path; int* kept; int* picked;
  long long ldt, ldd;
  int n_tokens, n_seqs, vocab, reserved;
};

__device__ __forceinline__ float vd_prob(float p) { return fminf(fmaxf(p, 0.f), 1.f); }     // (fmaxf drops what is no number)

// A clamped probability in 64 bits, times 2^-896: a float's bits moved into a double's, whose exponent has another offset.
// Exact, for zero and what is below the smallest normal number too; sums, differences and comparisons of such numbers need no
// scale.  (Conversions from 32 to 64 bits run at a quarter of the rate of the additions they feed.)
#define VD_SCALE 0x1p-896
__device__ __forceinline__ double vd_wide(float p) {
  const unsigned b = __float_as_uint(p);
  return __hiloint2double((int)(b >> 3), (int)(b << 29));
}
__device__ __forceinline__ double vd_lower(double p, double cover, double q) {
  const double w = fma(-cover, q, p);
  return __double2hiint(w) < 0 ? 0.0 : w;
}

struct VdSmem {
  int parent[VD_NODES], token[VD_NODES];
  float u[VD_NODES], p[VD_NODES], q[VD_NODES];   // a node's number, and its parent's probabilities of it
  double seg[VD_WARPS];                    // sums of the warps' stretches of the row, then running
  double told[2][16];                      // the blocks' sums, from everyone; every other sum has the other places
  int zeroed[VD_NODES];                    // ids the row has lost (looked up)
  double mass, cover;                      // (cover: 0 until the row has been lowered)
  int node, depth, n_zeroed, want;
  int last_lost;                           // the last id with any weight that the row has lost (looked up; 0: none)
  double all[16];                          // the blocks' sums, running
};

// What a walk costs is passes over a row, one behind the other: every rejection of a drawn child sums the lowered row before the
// next child can be tried, and the draw at the end sums it where that has not been done.  Measured: 64 trees of 9 to 16 nodes,
// 128,256 ids, drawn: 34 to 39 us (one pass over the 64 first rows and the draft's would be 10); a chain of six behind 128,256, in a
// replayed graph: 7.4 us, of which 3 are the dependent reads of the tree, its numbers and the row.
//
// W: ids of a load (4 where every row begins on 16 bytes); a warp has LINES loads of a row on their way together.
template <int W>
__global__ void __launch_bounds__(VD_THREADS, 2)
verify_drafts_kernel(const VerifyParams P) {
  constexpr int LINES = W == 4 ? 4 : 8, LINE = 32 * W;
  __shared__ VdSmem S;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_begun();
  pdl_wait();
  const int a = min(max(__ldcg(P.seq_start + b), 0), P.n_tokens), n = min(max(__ldcg(P.seq_start + b + 1), a), P.n_tokens) - a;
  if (n == 0) {                                    // (the same in the whole cluster)
    cluster_all_begun();
    if (c == 0 && tid == 0) { P.kept[b] = 0; P.picked[b] = -1; }
    return;
  }
  const int nodes = min(n, VD_NODES);
  for (int i = tid; i < nodes; i += VD_THREADS) {  // every node's numbers at once, whether the walk comes by or not
    const int parent = __ldcg(P.parents + a + i);
    int token = __ldcg(P.tokens + a + i);
    float p = 0.f, q = 0.f;
    if (parent >= 0 && parent < i && token >= 0 && token < P.vocab) {
      p = vd_prob(__ldcg(P.target + (long long)(a + parent) * P.ldt + token));
      q = P.draft ? vd_prob(__ldcg(P.draft + (long long)(a + parent) * P.ldd + token)) : 1.f;
    } else {
      token = -1;                                  // never taken, and the row stays as it is
    }
    S.parent[i] = parent; S.token[i] = token; S.u[i] = __ldcg(P.uniform + a + i); S.p[i] = p; S.q[i] = q;
  }
  if (tid == 0) { S.mass = 1.0; S.cover = 0.0; S.node = 0; S.depth = 0; S.n_zeroed = 0; S.last_lost = 0; }
  if (c == 0) for (int i = tid; i < n; i += VD_THREADS) P.path[a + i] = i == 0 ? 0 : -1;
  __syncthreads();
  cluster_all_begun();

  // A warp's stretch of the row, in whole lines of LINE ids.
  const int n_seg = C * VD_WARPS, lines = (P.vocab + LINE - 1) / LINE, per = (lines + n_seg - 1) / n_seg * LINE;
  const int seg = c * VD_WARPS + warp, s0 = (int)min((long long)seg * per, (long long)P.vocab), s1 = min(s0 + per, P.vocab);
  // this lane's ids i .. i + W - 1 of LINES lines from i on, of the target's row and, where it is to be lowered, the draft's
  auto fetch = [&](const float* trow, const float* drow, int i, int end, bool low, float (&p)[LINES][W], float (&q)[LINES][W]) {
#pragma unroll
    for (int x = 0; x < LINES; x++) {
      const int at = i + x * LINE;
#pragma unroll
      for (int e = 0; e < W; e++) p[x][e] = q[x][e] = 0.f;
      if (W == 4 && at + 3 < end) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(trow + at));
        p[x][0] = y.x; p[x][W / 4] = y.y; p[x][W / 2] = y.z; p[x][W - 1] = y.w;
        if (low) {
          const float4 z = __ldcg(reinterpret_cast<const float4*>(drow + at));
          q[x][0] = z.x; q[x][W / 4] = z.y; q[x][W / 2] = z.z; q[x][W - 1] = z.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < W; e++)
          if (at + e < end) { p[x][e] = __ldcg(trow + at + e); if (low) q[x][e] = __ldcg(drow + at + e); }
      }
    }
  };
  // d of W ids from i on, times VD_SCALE: the target's row, lowered by the draft's, without the ids it has lost (those of the
  // list that lie in this warp's stretch, if any do)
  auto weights = [&](float (&p)[W], float (&q)[W], int i, double cover, bool lost, double (&w)[W]) {
    unsigned most = 0;                             // (a number in [0, 1] has no larger bits than 1 has)
#pragma unroll
    for (int e = 0; e < W; e++) most = max(most, max(__float_as_uint(p[e]), __float_as_uint(q[e])));
    if (most > 0x3f800000u) {
#pragma unroll
      for (int e = 0; e < W; e++) { p[e] = vd_prob(p[e]); q[e] = vd_prob(q[e]); }
    }
#pragma unroll
    for (int e = 0; e < W; e++) w[e] = vd_wide(p[e]);
    if (cover > 0.0) {
#pragma unroll
      for (int e = 0; e < W; e++) w[e] = vd_lower(w[e], cover, vd_wide(q[e]));
    }
    if (lost) {
#pragma unroll 1
      for (int j = 0; j < S.n_zeroed; j++)
#pragma unroll
        for (int e = 0; e < W; e++) if (S.zeroed[j] == i + e) w[e] = 0.0;
    }
  };
  auto loses_between = [&](int from, int end) {
    bool mine = false;
    for (int j = lane; j < S.n_zeroed; j += 32) mine = mine || (S.zeroed[j] >= from && S.zeroed[j] < end);
    return __any_sync(0xffffffffu, mine) != 0;
  };
  auto sum_of = [&](const float* trow, const float* drow, double cover, int from, int end) {       // by one warp
    const bool lost = S.n_zeroed > 0 && loses_between(from, end);
    double sum = 0.0;
#pragma unroll 1
    for (int i0 = from; i0 < end; i0 += LINES * LINE) {
      float p[LINES][W], q[LINES][W];
      fetch(trow, drow, i0 + lane * W, end, cover > 0.0, p, q);
#pragma unroll
      for (int x = 0; x < LINES; x++) {
        double w[W];
        weights(p[x], q[x], i0 + x * LINE + lane * W, cover, lost, w);
        double part = 0.0;
#pragma unroll
        for (int e = 0; e < W; e++) part += w[e];
        sum += part;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };
  auto scan = [&](double v, int n) {               // running sums over the first n lanes
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d && lane < n) v += o;
    }
    return v;
  };
  // The walk is warp 0's in every block, with the same numbers and so the same way everywhere; where it needs the sum of a
  // row, all blocks work that out together.
  bool summed = false;                             // S.all holds the running sums of the row as it is (warp 0's)
  int last = 0, parity = 0;                        // the last child tried at this node (warp 0's)
  for (;;) {
    if (warp == 0) {
      int node = S.node, depth = S.depth, want = 0;
      while (!want) {
        int child = -1;                            // the next child of `node` behind `last`
        for (int i0 = last + 1; i0 < nodes && child < 0; i0 += 32) {
          const int i = i0 + lane;
          const unsigned have = __ballot_sync(0xffffffffu, i < nodes && S.parent[i] == node);
          if (have) child = i0 + __ffs(have) - 1;
        }
        if (child < 0) { want = summed ? 3 : 2; break; }
        last = child;
        const int token = S.token[child];
        if (token < 0) continue;
        const double mass = S.mass, q = P.draft ? vd_wide(S.q[child]) : VD_SCALE;
        double w = vd_wide(S.p[child]);
        if (S.cover > 0.0) w = vd_lower(w, S.cover, q);
        for (int j = 0; j < S.n_zeroed; j++) if (S.zeroed[j] == token) w = 0.0;
        __syncwarp();
        if (__dmul_rn(__dmul_rn((double)S.u[child], mass), q) < w) {
          node = child; depth++;                   // (its children come behind it)
          if (lane == 0) {
            if (c == 0) P.path[a + depth] = child;
            S.mass = 1.0; S.cover = 0.0; S.n_zeroed = 0; S.last_lost = 0;
          }
          summed = false;
        } else if (P.draft) {
          want = 1;
        } else {
          w *= 1.0 / VD_SCALE;
          if (lane == 0) {
            S.mass = mass - w > 0.0 ? mass - w : 0.0;
            S.zeroed[S.n_zeroed++] = token;
            if (w > 0.0) S.last_lost = token;
          }
          summed = false;
        }
        __syncwarp();
      }
      if (lane == 0) { S.node = node; S.depth = depth; S.want = want; }
    }
    __syncthreads();
    const int want = S.want;                       // 1: the sum of what a rejection leaves, 2: of the row as it is, 3: it is there
    if (want == 3) break;
    {
      const float* trow = P.target + (long long)(a + S.node) * P.ldt;
      const float* drow = P.draft ? P.draft + (long long)(a + S.node) * P.ldd : nullptr;
      const double cover = S.cover + (want == 1 ? S.mass : 0.0);
      const double sum = sum_of(trow, drow, cover, s0, s1);
      if (lane == 0) S.seg[warp] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      const double v = scan(lane < VD_WARPS ? S.seg[lane] : 0.0, VD_WARPS), total = __shfl_sync(0xffffffffu, v, VD_WARPS - 1);
      if (lane < VD_WARPS) S.seg[lane] = v;
      if (lane < C) cluster.map_shared_rank(&S, lane)->told[parity][c] = total;
    }
    cluster.sync();                                // (behind the last of these nothing of another block is touched)
    if (warp == 0) {
      const double v = scan(lane < C ? S.told[parity][lane] : 0.0, C), carry = __shfl_sync(0xffffffffu, v, C - 1);
      if (lane < C) S.all[lane] = v;
      summed = want == 2 || carry > 0.0;
      if (want == 1 && carry > 0.0 && lane == 0) { S.cover += S.mass; S.mass = carry * (1.0 / VD_SCALE); }      // (else the row stays as it was)
      __syncwarp();
    }
    parity ^= 1;
    if (want == 2) break;
  }
  // ---- the draw: the first block whose running sum is over the aim, in it the first warp's stretch, then, its lines shared out
  // among the warps, the first part of that, and the first id
  __syncthreads();                                 // (the blocks' sums are there)
  const double total = S.all[C - 1], aim = __dmul_rn((double)S.u[0], total);
  // the first of n lanes whose running sum is over the aim; none (rounding): the last one that has any weight
  auto find = [&](double v, double before, int n, bool& over) {
    const unsigned overs = __ballot_sync(0xffffffffu, lane < n && v > aim), anys = __ballot_sync(0xffffffffu, lane < n && v > before);
    over = overs != 0;
    return overs ? __ffs(overs) - 1 : anys ? 31 - __clz(anys) : 0;
  };
  bool crossed;
  const int block = find(lane < C ? S.all[lane] : 0.0, lane > 0 && lane < C ? S.all[lane - 1] : 0.0, C, crossed);
  if (c == 0 && tid == 0) {
    P.kept[b] = S.depth;
    if (!(total > 0.0)) P.picked[b] = S.last_lost; // nothing left to draw from: what was lost last, or 0
  }
  if (block != c || !(total > 0.0)) return;        // (the same in the whole block; nothing of another block is touched any more)
  const double front = c > 0 ? S.all[c - 1] : 0.0;
  const double mine = lane < VD_WARPS ? S.seg[lane] : 0.0, less = lane > 0 && lane < VD_WARPS ? S.seg[lane - 1] : 0.0;
  bool here;
  const int w_ = find(front + mine, front + less, VD_WARPS, here), found = c * VD_WARPS + w_;
  crossed = crossed && here;
  double base = front + (w_ > 0 ? S.seg[w_ - 1] : 0.0);
  const float* trow = P.target + (long long)(a + S.node) * P.ldt;
  const float* drow = P.draft ? P.draft + (long long)(a + S.node) * P.ldd : nullptr;
  const double cover = S.cover;
  const int f0 = (int)min((long long)found * per, (long long)P.vocab), f1 = min(f0 + per, P.vocab);
  const int part = (per / LINE + VD_WARPS - 1) / VD_WARPS * LINE;
  auto part_from = [&](int w) { return min(f0 + w * part, f1); };
  const double sum = sum_of(trow, drow, cover, part_from(warp), part_from(warp + 1));
  __syncthreads();                                 // (the stretches' sums are read)
  if (lane == 0) S.seg[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
  const double upto = scan(lane < VD_WARPS ? S.seg[lane] : 0.0, VD_WARPS);
  double before = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) before = 0.0;
  const int w2 = find(base + upto, base + before, VD_WARPS, here), g0 = part_from(w2), g1 = part_from(w2 + 1);
  crossed = crossed && here;
  base += __shfl_sync(0xffffffffu, before, w2);
  const bool lost = S.n_zeroed > 0 && loses_between(g0, g1);
  int pick = -1, positive = 0;
  for (int i0 = g0; i0 < g1 && pick < 0; i0 += LINES * LINE) {
    float p[LINES][W], q[LINES][W];
    fetch(trow, drow, i0 + lane * W, g1, cover > 0.0, p, q);
#pragma unroll
    for (int x = 0; x < LINES; x++) {
      if (i0 + x * LINE >= g1) break;
      const int i = i0 + x * LINE + lane * W;
      double w[W];
      weights(p[x], q[x], i, cover, lost, w);
      double v = 0.0;
#pragma unroll
      for (int e = 0; e < W; e++) v += w[e];
      double up = v;                               // running sums over the lanes
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += o;
      }
      double run = base + (up - v);
      int over = -1, any = -1;                     // this lane's first id over the aim, and last one with any weight
#pragma unroll
      for (int e = 0; e < W; e++) {
        run += w[e];
        if (w[e] > 0.0) { any = i + e; if (over < 0 && run > aim) over = i + e; }
      }
      const unsigned overs = __ballot_sync(0xffffffffu, over >= 0), anys = __ballot_sync(0xffffffffu, any >= 0);
      if (anys) positive = __shfl_sync(0xffffffffu, any, 31 - __clz(anys));
      if (overs && crossed && pick < 0) pick = __shfl_sync(0xffffffffu, over, __ffs(overs) - 1);
      base += __shfl_sync(0xffffffffu, up, 31);
    }
  }
  if (lane == 0) P.picked[b] = pick >= 0 ? pick : positive;
}

// (a property of the device and the kernel, and dear to ask for: kept for each device; an answer of none is not)
static int vd_resident(int C) {
  static std::atomic<int> known[64][5];            // clusters of 1, 2, 4, 8, 16
  int dev = 0, at = 0;
  while ((1 << at) < C) at++;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return resident_clusters((const void*)verify_drafts_kernel<4>, C, VD_THREADS);
  int n = known[dev][at].load(std::memory_order_relaxed);
  if (n == 0) {
    n = resident_clusters((const void*)verify_drafts_kernel<4>, C, VD_THREADS);
    known[dev][at].store(n, std::memory_order_relaxed);
  }
  return n;
}

// call: the parameters as the launcher packs them.
STRATUM_EXPORT int stratum_verify_drafts(const VerifyParams* call, cudaStream_t stream) {
  const VerifyParams P = *call;
  if (P.n_seqs <= 0) return 0;
  if (P.vocab < 1 || P.n_tokens < 0) return STRATUM_ERR_SHAPE;
  if (P.n_seqs > (1 << 26) || P.vocab > (1 << 30)) return STRATUM_ERR_LIMIT;
  const bool four = (((uintptr_t)P.target | (uintptr_t)P.draft) & 15) == 0 && P.ldt % 4 == 0 && P.ldd % 4 == 0;
  // As many blocks a row as leave every warp some lines of it, while all sequences' clusters find room at once (a cluster
  // lies within one part of the GPU: 37 clusters of eight do not, and took 17 us where 37 of four took 12)
  int C = 1;
  while (C < 16 && C * 2048 < P.vocab && P.n_seqs <= vd_resident(2 * C)) C *= 2;
  if (four) return launch_clusters<verify_drafts_kernel<4>>(P.n_seqs, C, VD_THREADS, stream, P);
  return launch_clusters<verify_drafts_kernel<1>>(P.n_seqs, C, VD_THREADS, stream, P);
}
