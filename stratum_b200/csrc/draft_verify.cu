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
// in the other blocks of the cluster.  Every thread takes its exponentials against the largest of its own values, so the
// blocks meet once: each tells the others its maximum (and where it is) and its sum against it, and a thread's values then
// need one factor.  (A row longer than sixteen blocks hold is read a second time.)
#define PR_THREADS 512
#define PR_HELD 32

struct Best { float v; int i; float sum; };        // the largest value, where it is first, sum of exp2((x - v) to_log2)
// Both together.  (A part without any value above -inf has the sum zero, and infinite values count one each.)
__device__ __forceinline__ Best both(Best a, Best b, float to_log2) {
  const bool second = b.v > a.v || (b.v == a.v && b.i < a.i);
  Best r = second ? b : a;
  const Best o = second ? a : b;
  r.sum += o.v == r.v ? o.sum : o.v == -INFINITY ? 0.f : o.sum * exp2f((o.v - r.v) * to_log2);
  return r;
}
__device__ __forceinline__ Best shfl_xor(Best b, int o) {
  return Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o), __shfl_xor_sync(0xffffffffu, b.sum, o)};
}

// W: values of a load and a store (4 where every row begins on 16 bytes)
template <bool HELD, int W>
__global__ void __launch_bounds__(PR_THREADS, 2)
token_probs_kernel(const float* logits, long long ld, const float* temperature, float* out, long long ldo, int vocab, int slice) {
  __shared__ Best parts[PR_THREADS / 32], blocks[16];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int i0 = min(c * slice, vocab), n = min(vocab - i0, slice);
  const float* in = logits + row * ld + i0;
  float* to = out + row * ldo + i0;
  const float t = ld_fresh(temperature + row);
  const bool greedy = !(t > 0.f);
  const float to_log2 = greedy ? 0.f : 1.4426950408889634f / t;
  auto clean = [](float v) { return v == v ? v : -INFINITY; };
  // against `m`, no less than v: 1 at the maximum (infinite ones too), 0 at -inf
  auto weight = [&](float v, float m) { return v == m ? 1.f : v == -INFINITY ? 0.f : exp2f((v - m) * to_log2); };
  float x[HELD ? PR_HELD : 1];
  Best b{-INFINITY, 0x7fffffff, 0.f};
  auto place = [&](int k) { return ((k / W) * PR_THREADS + tid) * W + k % W; };      // of a thread's k-th value in the slice
  if (HELD) {
#pragma unroll
    for (int k = 0; k < PR_HELD; k += W) {
      const int i = place(k);
      if (W == 4 && i + 3 < n) {
        const float4 v = ld_fresh(reinterpret_cast<const float4*>(in + i));
        x[k] = v.x; x[k + W / 4] = v.y; x[k + W / 2] = v.z; x[k + W - 1] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < W; e++) x[k + e] = i + e < n ? ld_fresh(in + i + e) : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) { x[k] = clean(x[k]); if (x[k] > b.v) { b.v = x[k]; b.i = i0 + place(k); } }
    if (b.v != -INFINITY) {
#pragma unroll
      for (int k = 0; k < PR_HELD; k++) { x[k] = weight(x[k], b.v); b.sum += x[k]; }
    }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) {
      const float v = clean(ld_fresh(in + i));
      if (v > b.v) {
        b.sum = b.v == -INFINITY ? 0.f : b.sum * exp2f((b.v - v) * to_log2);
        b.v = v; b.i = i0 + i;
      }
      if (v != -INFINITY) b.sum += weight(v, b.v);
    }
  }
  const float mine = b.v;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) b = both(b, shfl_xor(b, o), to_log2);
  if (lane == 0) parts[warp] = b;
  __syncthreads();
  if (warp == 0) {
    b = parts[lane % (PR_THREADS / 32)];
#pragma unroll
    for (int o = PR_THREADS / 64; o > 0; o >>= 1) b = both(b, shfl_xor(b, o), to_log2);
    if (lane < C) *cluster.map_shared_rank(&blocks[c], lane) = b;
  }
  cluster.sync();                                  // (nothing of another block is touched behind it)
  b = blocks[0];
  for (int i = 1; i < C; i++) b = both(b, blocks[i], to_log2);
  if (greedy || b.v == -INFINITY) {                // (the same in the whole cluster)
    const int best = b.v == -INFINITY ? -1 : b.i - i0;
    for (int i = tid; i < n; i += PR_THREADS) to[i] = i == best ? 1.f : 0.f;
    return;
  }
  const float inv = 1.0f / b.sum;
  if (HELD) {
    const float f = mine == -INFINITY ? 0.f : weight(mine, b.v) * inv;
#pragma unroll
    for (int k = 0; k < PR_HELD; k++) x[k] = mine == -INFINITY ? 0.f : x[k] * f;
#pragma unroll
    for (int k = 0; k < PR_HELD; k += W) {
      const int i = place(k);
      if (W == 4 && i + 3 < n) {
        *reinterpret_cast<float4*>(to + i) = make_float4(x[k], x[k + W / 4], x[k + W / 2], x[k + W - 1]);
      } else {
#pragma unroll
        for (int e = 0; e < W; e++) if (i + e < n) to[i + e] = x[k + e];
      }
    }
  } else {
    for (int i = tid; i < n; i += PR_THREADS) to[i] = weight(clean(ld_fresh(in + i)), b.v) * inv;
  }
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
  const int slice = (((vocab + C - 1) / C) + 3) & ~3;
  const bool four = (((uintptr_t)logits | (uintptr_t)out) & 15) == 0 && (rows == 1 || (ld % 4 == 0 && ldo % 4 == 0));
  if (slice <= PR_THREADS * PR_HELD) {
    if (four) return launch_clusters<token_probs_kernel<true, 4>>(rows, C, PR_THREADS, stream, logits, ld, temperature, out, ldo, vocab, slice);
    return launch_clusters<token_probs_kernel<true, 1>>(rows, C, PR_THREADS, stream, logits, ld, temperature, out, ldo, vocab, slice);
  }
  return launch_clusters<token_probs_kernel<false, 1>>(rows, C, PR_THREADS, stream, logits, ld, temperature, out, ldo, vocab, slice);
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

struct VdSmem {
  int parent[VD_NODES], token[VD_NODES];
  float u[VD_NODES], p[VD_NODES], q[VD_NODES];   // a node's number, and its parent's probabilities of it
  double seg[2][VD_WARPS];                 // sums of the warps' stretches of the row; every other sum has the other array
  double masses[VD_NODES];                 // the masses the row has been lowered at
  int zeroed[VD_NODES];                    // ids the row has lost (looked up)
  double mass;
  int node, depth, n_masses, n_zeroed, want;
  double all[16 * VD_WARPS];               // the whole cluster's sums, running
};

__global__ void __launch_bounds__(VD_THREADS, 2)
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
  // d at eight places 32 apart, from i on: the target's row, lowered at k masses, without the ids it has lost (those of the
  // list that lie in this warp's stretch, if any do)
  auto weights = [&](const float* trow, const float* drow, int i, int end, int k, bool lost, double (&w)[8]) {
    float p[8], q[8];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      p[x] = i + 32 * x < end ? __ldcg(trow + i + 32 * x) : 0.f;
      q[x] = i + 32 * x < end && k > 0 ? __ldcg(drow + i + 32 * x) : 0.f;
    }
#pragma unroll
    for (int x = 0; x < 8; x++) w[x] = (double)vd_prob(p[x]);
    if (k > 0) {
      double qd[8];
#pragma unroll
      for (int x = 0; x < 8; x++) qd[x] = (double)vd_prob(q[x]);
#pragma unroll 1
      for (int j = 0; j < k; j++) {
        const double m = S.masses[j];
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const double y = __dsub_rn(w[x], __dmul_rn(m, qd[x]));
          w[x] = y > 0.0 ? y : 0.0;
        }
      }
    }
    if (lost) {
#pragma unroll 1
      for (int j = 0; j < S.n_zeroed; j++)
#pragma unroll
        for (int x = 0; x < 8; x++) if (S.zeroed[j] == i + 32 * x) w[x] = 0.0;
    }
  };
  auto loses_between = [&](int from, int end) {
    bool mine = false;
    for (int j = lane; j < S.n_zeroed; j += 32) mine = mine || (S.zeroed[j] >= from && S.zeroed[j] < end);
    return __any_sync(0xffffffffu, mine) != 0;
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
        const double mass = S.mass, q = (double)S.q[child];              // (looked up: q = 1)
        double w = (double)S.p[child];
        for (int j = 0; j < S.n_masses; j++) { w = __dsub_rn(w, __dmul_rn(S.masses[j], q)); w = w > 0.0 ? w : 0.0; }
        for (int j = 0; j < S.n_zeroed; j++) if (S.zeroed[j] == token) w = 0.0;
        __syncwarp();
        if (__dmul_rn(__dmul_rn((double)S.u[child], mass), q) < w) {
          node = child; depth++;                   // (its children come behind it)
          if (lane == 0) {
            if (c == 0) P.path[a + depth] = child;
            S.mass = 1.0; S.n_masses = 0; S.n_zeroed = 0;
          }
          summed = false;
        } else if (P.draft) {
          if (lane == 0) S.masses[S.n_masses] = mass;
          want = 1;
        } else {
          if (lane == 0) { S.mass = mass - w > 0.0 ? mass - w : 0.0; S.zeroed[S.n_zeroed++] = token; }
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
      const int k = S.n_masses + (want == 1 ? 1 : 0);
      const bool lost = S.n_zeroed > 0 && loses_between(s0, s1);
      double sum = 0.0;
#pragma unroll 1
      for (int i0 = s0; i0 < s1; i0 += 32 * 8) {
        double w[8];
        weights(trow, drow, i0 + lane, s1, k, lost, w);
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) S.seg[parity][warp] = sum;
    }
    cluster.sync();
    if (warp == 0) {                               // running sums over all stretches of the cluster, in order
      double carry = 0.0;
      for (int i0 = 0; i0 < n_seg; i0 += 32) {
        const int i = i0 + lane;
        double v = i < n_seg ? cluster.map_shared_rank(&S, i / VD_WARPS)->seg[parity][i % VD_WARPS] : 0.0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(0xffffffffu, v, d);
          if (lane >= d) v += o;
        }
        if (i < n_seg) S.all[i] = carry + v;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
      summed = want == 2 || carry > 0.0;
      if (want == 1 && carry > 0.0 && lane == 0) { S.mass = carry; S.n_masses++; }      // (else the row stays as it was)
      __syncwarp();
    }
    parity ^= 1;
    if (want == 2) break;
  }
  // ---- the draw
  if (warp == 0) {
    const double total = S.all[n_seg - 1], aim = __dmul_rn((double)S.u[0], total);
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
    int pick = -1, positive = 0;
    if (found / VD_WARPS == c && total > 0.0) {
      const float* trow = P.target + (long long)(a + S.node) * P.ldt;
      const float* drow = P.draft ? P.draft + (long long)(a + S.node) * P.ldd : nullptr;
      const int f0 = min(found * per * 32, P.vocab), f1 = min(f0 + per * 32, P.vocab);
      const bool lost = S.n_zeroed > 0 && loses_between(f0, f1);
      double base = found > 0 ? S.all[found - 1] : 0.0;
      for (int i0 = f0; i0 < f1 && pick < 0; i0 += 32 * 8) {
        double w[8];
        weights(trow, drow, i0 + lane, f1, S.n_masses, lost, w);
#pragma unroll
        for (int x = 0; x < 8; x++) {
          double v = w[x];
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += o;
          }
          const unsigned over = __ballot_sync(0xffffffffu, w[x] > 0.0 && base + v > aim);
          const unsigned any = __ballot_sync(0xffffffffu, w[x] > 0.0);
          if (any) positive = i0 + 32 * x + 31 - __clz(any);
          if (crossed && over && pick < 0) pick = i0 + 32 * x + __ffs(over) - 1;
          base += __shfl_sync(0xffffffffu, v, 31);
        }
      }
      if (lane == 0) P.picked[b] = pick >= 0 ? pick : positive;
    }
    if (c == 0 && lane == 0) {
      P.kept[b] = S.depth;
      if (!(total > 0.0)) P.picked[b] = 0;         // nothing to draw from
    }
  }
  cluster.sync();                                  // nobody leaves while its sums may still be read
}

// call: the parameters as the launcher packs them.
STRATUM_EXPORT int stratum_verify_drafts(const VerifyParams* call, cudaStream_t stream) {
  const VerifyParams P = *call;
  if (P.n_seqs <= 0) return 0;
  if (P.vocab < 1 || P.n_tokens < 0) return STRATUM_ERR_SHAPE;
  if (P.n_seqs > (1 << 26) || P.vocab > (1 << 30)) return STRATUM_ERR_LIMIT;
  // as many blocks a row as leave every warp a few lines of it and all of them resident (two to an SM)
  int C = 1;
  while (C < 16 && C * 2048 < P.vocab && (long long)P.n_seqs * C * 2 <= 2 * sms()) C *= 2;
  return launch_clusters<verify_drafts_kernel>(P.n_seqs, C, VD_THREADS, stream, P);
}
