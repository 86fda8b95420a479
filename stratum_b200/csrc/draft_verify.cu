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
//     and mass = sum d, unless nothing would be left;
//   looked up, without a distribution:  taken if u mass < d(x);  else  mass = max(mass - d(x), 0) and d(x) = 0.
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

#include "common.cuh"

namespace cg = cooperative_groups;

static int sms() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
  }
  return n;
}

// rows clusters of `cluster` blocks each
template <auto kernel, typename... Args>
static int launch_clusters(unsigned rows, unsigned cluster, unsigned threads, cudaStream_t stream, Args... args) {
  static unsigned long long done = 0;              // devices on which this kernel may have clusters of sixteen
  int dev = 0;
  cudaGetDevice(&dev);
  if (cluster > 8 && !(done & (1ull << (dev & 63)))) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
    done |= 1ull << (dev & 63);
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

// ================================================================ probabilities
// A row is read once and written once: its values stay in registers, 32 to a thread, 16,384 to a block, the rest of the row
// in the other blocks of the cluster.  (A row longer than 16 blocks hold is read again for every stage.)
#define PR_THREADS 512
#define PR_HELD 32

struct Best { float v; int i; };
__device__ __forceinline__ Best best_of(Best a, Best b) { return (b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a; }

// The cluster's maximum (with the lowest index that has it) or sum, the same in every thread.
struct PrSmem { Best best[17]; float sum[17]; Best all_best; float all_sum; };

template <bool HELD>
__global__ void __launch_bounds__(PR_THREADS, 2)
token_probs_kernel(const float* logits, long long ld, const float* temperature, float* out, long long ldo, int vocab) {
  __shared__ PrSmem S;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int slice = (vocab + C - 1) / C, i0 = c * slice, n = max(min(vocab - i0, slice), 0);
  const float* in = logits + row * ld + i0;
  float* to = out + row * ldo + i0;
  float x[HELD ? PR_HELD : 1];
  auto read = [&](int i) { const float v = ld_fresh(in + i); return v == v ? v : -INFINITY; };
  Best b{-INFINITY, 0x7fffffff};
  if (HELD) {
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) { const int i = k * PR_THREADS + tid; x[k] = i < n ? read(i) : -INFINITY; }
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) if (x[k] > b.v) { b.v = x[k]; b.i = i0 + k * PR_THREADS + tid; }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) { const float v = read(i); if (v > b.v) { b.v = v; b.i = i0 + i; } }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    b = best_of(b, Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)});
  if (lane == 0) S.best[warp] = b;
  __syncthreads();
  if (warp == 0) {
    b = lane < PR_THREADS / 32 ? S.best[lane] : Best{-INFINITY, 0x7fffffff};
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      b = best_of(b, Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)});
    if (lane == 0) S.best[16] = b;
  }
  cluster.sync();
  if (warp == 0) {
    b = lane < C ? cluster.map_shared_rank(&S, lane)->best[16] : Best{-INFINITY, 0x7fffffff};
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      b = best_of(b, Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)});
    if (lane == 0) S.all_best = b;
  }
  __syncthreads();
  const float m = S.all_best.v, t = ld_fresh(temperature + row);
  if (!(t > 0.f) || m == -INFINITY) {              // (the same in the whole cluster)
    const int best = m == -INFINITY ? -1 : S.all_best.i - i0;
    for (int i = tid; i < n; i += PR_THREADS) to[i] = i == best ? 1.f : 0.f;
    cluster.sync();                                // nobody leaves while its maximum may still be read
    return;
  }
  const float to_log2 = 1.4426950408889634f / t;
  auto weight = [&](float v) { return v == m ? 1.f : v == -INFINITY ? 0.f : exp2f((v - m) * to_log2); };
  float sum = 0.f;
  if (HELD) {
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) { x[k] = weight(x[k]); sum += x[k]; }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) sum += weight(read(i));
  }
  sum = warp_sum(sum);
  if (lane == 0) S.sum[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = warp_sum(lane < PR_THREADS / 32 ? S.sum[lane] : 0.f);
    if (lane == 0) S.sum[16] = sum;
  }
  cluster.sync();
  if (warp == 0) {
    sum = warp_sum(lane < C ? cluster.map_shared_rank(&S, lane)->sum[16] : 0.f);
    if (lane == 0) S.all_sum = sum;
  }
  __syncthreads();
  const float inv = 1.0f / S.all_sum;
  if (HELD) {
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) { const int i = k * PR_THREADS + tid; if (i < n) to[i] = x[k] * inv; }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) to[i] = weight(read(i)) * inv;
  }
  cluster.sync();
}

// logits float32 [rows][ld], temperature float32 [rows], out float32 [rows][ldo]; out may be logits (the same rows at the same
// distance).
STRATUM_EXPORT int stratum_token_probs(const float* logits, long long ld, const float* temperature, float* out, long long ldo,
                                       int rows, int vocab, cudaStream_t stream) {
  if (rows <= 0 || vocab <= 0) return 0;
  if (rows > (1 << 26) || vocab > (1 << 30)) return STRATUM_ERR_LIMIT;
  // enough blocks to hold a row; beyond that, where a few rows leave the GPU empty, blocks of shorter slices
  int C = 1;
  while (C < 16 && ((long long)C * PR_THREADS * PR_HELD < vocab || (C * 4096 < vocab && (long long)rows * C * 2 <= sms()))) C *= 2;
  if ((long long)C * PR_THREADS * PR_HELD >= vocab)
    return launch_clusters<token_probs_kernel<true>>(rows, C, PR_THREADS, stream, logits, ld, temperature, out, ldo, vocab);
  return launch_clusters<token_probs_kernel<false>>(rows, C, PR_THREADS, stream, logits, ld, temperature, out, ldo, vocab);
}

// ================================================================ verification
#define VD_THREADS 512
#define VD_WARPS (VD_THREADS / 32)
#define VD_NODES 1024            // nodes of a sequence that are looked at

struct VerifyParams {
  const float* target; long long ldt;
  const float* draft; long long ldd;       // null: looked up
  const int* tokens; const int* parents; const int* seq_start; const float* uniform;
  int* path; int* kept; int* picked;
  int n_tokens, n_seqs, vocab;
};

__device__ __forceinline__ float vd_prob(float p) { return fminf(fmaxf(p, 0.f), 1.f); }     // (fmaxf drops what is no number)

struct VdSmem {
  int parent[VD_NODES], token[VD_NODES];
  float u[VD_NODES], p[VD_NODES], q[VD_NODES];   // a node's number, and its parent's probabilities of it
  double seg[VD_WARPS];                    // sums of the warps' stretches of the row
  double masses[VD_NODES];                 // the masses the row has been lowered at
  int zeroed[VD_NODES];                    // ids the row has lost (looked up)
  double mass;
  int node, depth, n_masses, n_zeroed, want;     // want: 1 the sum of what a rejection leaves, 2 of the row as it is
  double all[16 * VD_WARPS];               // the whole cluster's sums, running
};

__global__ void __launch_bounds__(VD_THREADS)
verify_drafts_kernel(const VerifyParams P) {
  __shared__ VdSmem S;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int a = min(max(__ldcg(P.seq_start + b), 0), P.n_tokens), n = min(max(__ldcg(P.seq_start + b + 1), a), P.n_tokens) - a;
  if (n == 0) {                                    // (the same in the whole cluster)
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
  if (tid == 0) { S.mass = 1.0; S.node = 0; S.depth = 0; S.n_masses = 0; S.n_zeroed = 0; }
  if (c == 0) for (int i = tid; i < n; i += VD_THREADS) P.path[a + i] = i == 0 ? 0 : -1;
  __syncthreads();

  // A warp's stretch of the row, in whole lines of 32.
  const int n_seg = C * VD_WARPS, lines = (P.vocab + 31) / 32, per = (lines + n_seg - 1) / n_seg;
  const int seg = c * VD_WARPS + warp, s0 = min(seg * per * 32, P.vocab), s1 = min(s0 + per * 32, P.vocab);
  // d(i): the target's row, lowered at k masses, without the ids it has lost
  auto weight = [&](float p, float q, int i, int k, bool lost) -> double {
    double w = (double)vd_prob(p);
    if (k > 0) {
      const double qd = (double)vd_prob(q);
      for (int j = 0; j < k; j++) { w = __dsub_rn(w, __dmul_rn(S.masses[j], qd)); w = w > 0.0 ? w : 0.0; }
    }
    if (lost) for (int j = 0; j < S.n_zeroed; j++) if (S.zeroed[j] == i) w = 0.0;
    return w;
  };
  auto loses_here = [&]() {                        // whether this warp's stretch has lost any id
    bool mine = false;
    for (int j = lane; j < S.n_zeroed; j += 32) mine = mine || (S.zeroed[j] >= s0 && S.zeroed[j] < s1);
    return __any_sync(0xffffffffu, mine);
  };
  bool summed = false;                             // S.all holds the running sums of the row as it is
  int last = 0;                                    // the last child tried at this node (warp 0's)
  for (;;) {
    // ---- the walk, by warp 0 of every block alike, until a sum over a row is needed
    if (warp == 0) {
      int node = S.node, depth = S.depth, want = 0;
      while (!want) {
        // the next child of `node` behind `last`
        int child = -1;
        for (int i0 = last + 1; i0 < nodes && child < 0; i0 += 32) {
          const int i = i0 + lane;
          const unsigned have = __ballot_sync(0xffffffffu, i < nodes && S.parent[i] == node);
          if (have) child = i0 + __ffs(have) - 1;
        }
        if (child < 0) { want = 2; break; }
        last = child;
        const int token = S.token[child];
        const float u = S.u[child], p = S.p[child], q = S.q[child];
        if (token < 0) continue;
        const double w = weight(p, q, token, S.n_masses, true), mass = S.mass;
        if (__dmul_rn(__dmul_rn((double)u, mass), (double)q) < w) {          // (looked up: q = 1)
          node = child; depth++;
          if (c == 0 && lane == 0) P.path[a + depth] = child;
          __syncwarp();
          if (lane == 0) { S.mass = 1.0; S.n_masses = 0; S.n_zeroed = 0; }
          __syncwarp();
          summed = false;
          last = child;                            // (children come behind their parents)
        } else if (P.draft) {
          __syncwarp();
          if (lane == 0) S.masses[S.n_masses] = mass;
          __syncwarp();
          want = 1;
        } else {
          __syncwarp();
          if (lane == 0) {
            S.mass = mass - w > 0.0 ? mass - w : 0.0;
            S.zeroed[S.n_zeroed++] = token;
          }
          __syncwarp();
          summed = false;
        }
      }
      if (lane == 0) { S.node = node; S.depth = depth; S.want = want; if (want == 2 && summed) S.want = 3; }
    }
    __syncthreads();
    const int want = S.want;
    if (want == 3) break;                            // the sums of the last rejection are those of the row as it is
    // ---- the sums of the stretches
    const float* trow = P.target + (long long)(a + S.node) * P.ldt;
    const float* drow = P.draft ? P.draft + (long long)(a + S.node) * P.ldd : nullptr;
    const int k = S.n_masses + (want == 1 ? 1 : 0);
    {
      double sum = 0.0;
      const bool lost = S.n_zeroed > 0 && loses_here();
#pragma unroll 1
      for (int i0 = s0; i0 < s1; i0 += 32 * 8) {
        float p[8], q[8];
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const int i = i0 + 32 * x + lane;
          p[x] = i < s1 ? __ldcg(trow + i) : 0.f;
          q[x] = i < s1 && k > 0 ? __ldcg(drow + i) : 0.f;
        }
#pragma unroll
        for (int x = 0; x < 8; x++) sum += weight(p[x], q[x], i0 + 32 * x + lane, k, lost);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) S.seg[warp] = sum;
    }
    cluster.sync();
    if (warp == 0) {                                 // running sums over all stretches of the cluster, in order
      double carry = 0.0;
      for (int i0 = 0; i0 < n_seg; i0 += 32) {
        const int i = i0 + lane;
        double v = i < n_seg ? cluster.map_shared_rank(&S, i / VD_WARPS)->seg[i % VD_WARPS] : 0.0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(0xffffffffu, v, d);
          if (lane >= d) v += o;
        }
        if (i < n_seg) S.all[i] = carry + v;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
      __syncwarp();
    }
    cluster.sync();                                  // (the sums have been read; S.all is there)
    if (want == 2) break;
    const double left = S.all[n_seg - 1];
    summed = left > 0.0;
    __syncthreads();
    if (tid == 0 && left > 0.0) { S.mass = left; S.n_masses++; }       // (else the row stays as it was)
    __syncthreads();
  }
  // ---- the draw
  const double total = S.all[n_seg - 1], aim = __dmul_rn((double)S.u[0], total);
  if (c == 0 && tid == 0) {
    P.kept[b] = S.depth;
    if (!(total > 0.0)) P.picked[b] = 0;             // nothing to draw from
  }
  if (!(total > 0.0)) return;
  if (warp != 0) return;
  // the first stretch whose running sum is over the aim; none (rounding): the last one that has any weight
  int found = -1, last_any = 0;
  for (int i0 = 0; i0 < n_seg; i0 += 32) {
    const int i = i0 + lane;
    const double v = i < n_seg ? S.all[i] : 0.0, before = i > 0 && i < n_seg ? S.all[i - 1] : 0.0;
    const unsigned over = __ballot_sync(0xffffffffu, i < n_seg && v > aim);
    const unsigned any = __ballot_sync(0xffffffffu, i < n_seg && v > before);
    if (over && found < 0) found = i0 + __ffs(over) - 1;
    if (any) last_any = i0 + 31 - __clz(any);
  }
  const bool crossed = found >= 0;
  if (!crossed) found = last_any;
  if (found / VD_WARPS != c) return;
  const float* trow = P.target + (long long)(a + S.node) * P.ldt;
  const float* drow = P.draft ? P.draft + (long long)(a + S.node) * P.ldd : nullptr;
  const int f0 = min(found * per * 32, P.vocab), f1 = min(f0 + per * 32, P.vocab), k = S.n_masses;
  double base = found > 0 ? S.all[found - 1] : 0.0;
  int pick = -1, positive = f0;
  for (int i0 = f0; i0 < f1 && pick < 0; i0 += 32 * 8) {
    float p[8], q[8];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      const int i = i0 + 32 * x + lane;
      p[x] = i < f1 ? __ldcg(trow + i) : 0.f;
      q[x] = i < f1 && k > 0 ? __ldcg(drow + i) : 0.f;
    }
#pragma unroll
    for (int x = 0; x < 8; x++) {
      const int i = i0 + 32 * x + lane;
      const double w = i < f1 ? weight(p[x], q[x], i, k, true) : 0.0;
      double v = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
      }
      const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && base + v > aim);
      const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
      if (any) positive = i0 + 32 * x + 31 - __clz(any);
      if (crossed && over && pick < 0) pick = i0 + 32 * x + __ffs(over) - 1;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  if (lane == 0) P.picked[b] = pick >= 0 ? pick : positive;
}

STRATUM_EXPORT int stratum_verify_drafts(const float* target, long long ldt, const float* draft, long long ldd, const int* tokens,
                                         const int* parents, const int* seq_start, const float* uniform, int* path, int* kept,
                                         int* picked, int n_tokens, int n_seqs, int vocab, cudaStream_t stream) {
  if (n_seqs <= 0) return 0;
  if (vocab < 1 || n_tokens < 0) return STRATUM_ERR_SHAPE;
  if (n_seqs > (1 << 26) || vocab > (1 << 30)) return STRATUM_ERR_LIMIT;
  VerifyParams P;
  P.target = target; P.ldt = ldt; P.draft = draft; P.ldd = ldd;
  P.tokens = tokens; P.parents = parents; P.seq_start = seq_start; P.uniform = uniform;
  P.path = path; P.kept = kept; P.picked = picked;
  P.n_tokens = n_tokens; P.n_seqs = n_seqs; P.vocab = vocab;
  int C = 1;
  while (C < 16 && C * 2048 < vocab && (C < 8 || (long long)n_seqs * C * 2 <= 2 * sms())) C *= 2;
  return launch_clusters<verify_drafts_kernel>(n_seqs, C, VD_THREADS, stream, P);
}
