// Drafted tokens against the target's probabilities: draft i stands while u_i q_i(x_i) < p_i(x_i); the token after the last
// that stands is drawn from max(p - q, 0) there (from p behind the last draft) by the inverse of the distribution.
#include <math.h>

#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"
#include "umma.cuh"

namespace dion {

namespace {

constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 8;  // CTAs of a sequence

__device__ __forceinline__ double usable(double w) { return w > 0.0 && w < INFINITY ? w : 0.0; }

// the value of `v` in CTA `rank` of the cluster
__device__ __forceinline__ double remote(const double* v, int rank) {
  const uint32_t at = mapa_shared(smem_u32(v), (uint32_t)rank);
  double r;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(r) : "r"(at) : "memory");
  return r;
}

// A cluster of eight CTAs per sequence, each with an eighth of the vocabulary: the weights' sums go over the cluster's shared memory,
// and the CTA in whose eighth the border lies finds the token.  Reads one row of either distribution; 64 sequences of 128256 tokens,
// of which that is 66 MB, are bound by memory, a single one by the latencies of its chain: drafts, weights, sums, search.
//
// Weights are differences of fp32 values in 64 bits and so are their sums, whose order then decides nothing: two orders differ by some
// 1e-16 of the whole, the border that a draw has to hit to tell them apart.
//
// A warp takes consecutive tokens, 32 x 4 at a time (16 bytes a lane where the rows allow), so that the search goes down from the
// CTA's sum over the warps' to one warp, which alone goes through its tokens again.
template <int V>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyDrafts p) {
  __shared__ double warp_sum[2][kVerifyWarps + 1];  // of the differences and of the row itself; the CTA's in the end
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / kVerifyCluster, rank = blockIdx.x % kVerifyCluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long* tokens = p.tokens + b * p.tokens_seq;
  const float* u = p.uniforms + b * p.uniforms_seq;
  // the first draft that falls, a lane for each
  int a = p.drafts;
  long long x = -1;
  for (int base = 0; base < p.drafts; base += 32) {
    const int i = base + lane;
    bool falls = false, known = true;
    long long mine = -1;
    if (i < p.drafts) {
      mine = tokens[i];
      known = mine >= 0 && mine < p.vocab;
      falls = true;
      if (known) {
        const double q = p.draft ? (double)p.draft[b * p.draft_seq + i * p.draft_row + mine] : 1.0;
        falls = !((double)u[i] * q < (double)p.target[b * p.target_seq + i * p.target_row + mine]);
      }
    }
    if (!known && rank == 0 && warp == 0) bad_argument(p.status);
    const unsigned at = __ballot_sync(0xffffffffu, falls);
    if (at) {
      const int first = __ffs(at) - 1;
      a = base + first;
      x = __shfl_sync(0xffffffffu, mine, first);  // one outside the vocabulary is no token's
      break;
    }
  }
  const bool all = a == p.drafts;
  const float* row = p.target + b * p.target_seq + a * p.target_row;
  const float* minus = p.draft && !all ? p.draft + b * p.draft_seq + a * p.draft_row : nullptr;
  const long long certain = !p.draft && !all ? x : -1;  // the draft's only token

  // V tokens of a lane: the differences and the row's own values
  auto weights = [&](int i, double (&d)[V], double (&w)[V]) {
    float t[V], q[V];
    if constexpr (V == 4) {
      const float4 r4 = i < p.vocab ? *reinterpret_cast<const float4*>(row + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 q4 = minus && i < p.vocab ? *reinterpret_cast<const float4*>(minus + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      t[0] = r4.x, t[1] = r4.y, t[2] = r4.z, t[3] = r4.w;
      q[0] = q4.x, q[1] = q4.y, q[2] = q4.z, q[3] = q4.w;
    } else {
      t[0] = i < p.vocab ? row[i] : 0.f;
      q[0] = minus && i < p.vocab ? minus[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      w[k] = usable(t[k]);
      d[k] = usable((double)t[k] - (i + k == certain ? 1.0 : (double)q[k]));
    }
  };
  // tokens of this warp: `per` rounds of 32 * V
  constexpr int round = 32 * V, everybody = kVerifyCluster * kVerifyWarps * round;
  const int per = (int)(((long long)p.vocab + everybody - 1) / everybody);
  const long long begin = ((long long)rank * kVerifyWarps + warp) * per * round;
  double left = 0.0, whole = 0.0;
#pragma unroll 4
  for (int r = 0; r < per; ++r) {
    const long long i = begin + r * round + lane * V;
    if (i < p.vocab) {
      double d[V], w[V];
      weights((int)i, d, w);
#pragma unroll
      for (int k = 0; k < V; ++k) left += d[k], whole += w[k];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    left += __shfl_xor_sync(0xffffffffu, left, o);
    whole += __shfl_xor_sync(0xffffffffu, whole, o);
  }
  if (lane == 0) warp_sum[0][warp] = left, warp_sum[1][warp] = whole;
  __syncthreads();
  if (threadIdx.x < 2) {
    double s = 0.0;
    for (int i = 0; i < kVerifyWarps; ++i) s += warp_sum[threadIdx.x][i];
    warp_sum[threadIdx.x][kVerifyWarps] = s;
  }
  cluster_sync_all();
  // which distribution, its sum, and what lies before this CTA
  int which = all ? 1 : 0;
  double total, before;
  for (;; which = 1) {
    const double mine = lane < kVerifyCluster ? remote(&warp_sum[which][kVerifyWarps], lane) : 0.0;
    total = before = 0.0;
    for (int i = 0; i < kVerifyCluster; ++i) {
      const double s = __shfl_sync(0xffffffffu, mine, i);
      if (i < rank) before += s;
      total += s;
    }
    if (total > 0.0 || which == 1) break;  // p - q leaves nothing: p itself
  }
  // The token is the first whose running sum exceeds the border.  The sums before a CTA are added up in one order by all of them, and
  // those before a warp by all warps of its CTA; each of the two takes what lies before the next one's start, the last warp the rest,
  // so that exactly one warp looks, wherever roundings put the border.
  const double border = (double)u[p.drafts] * total;
  if (rank == 0 && threadIdx.x == 0) {
    p.accepted[b] = a;
    if (!(total > 0.0) || !(border < total)) p.token[b] = total > 0.0 && border >= total ? p.vocab - 1 : 0;  // the latter: a uniform that is none
  }
  const bool here = total > 0.0 && border < total && (rank == 0 || before <= border) &&
                    (rank == kVerifyCluster - 1 || before + warp_sum[which][kVerifyWarps] > border);
  for (int i = 0; i < warp; ++i) before += warp_sum[which][i];
  if (here && (warp == 0 || before <= border) && (warp == kVerifyWarps - 1 || before + warp_sum[which][warp] > border)) {
    double run = before;
    bool found = false;
    for (int r = 0; r < per && !found; ++r) {
      const long long i = begin + r * round + lane * V;
      double d[V], w[V], mine = 0.0;
#pragma unroll
      for (int k = 0; k < V; ++k) d[k] = w[k] = 0.0;
      if (i < p.vocab) weights((int)i, d, w);
#pragma unroll
      for (int k = 0; k < V; ++k) mine += which ? w[k] : d[k];
      double upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
      }
      const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && run + upto > border);
      found = over != 0;
      if (found && lane == __ffs(over) - 1) {
        double s = run + upto - mine;
        long long token = i;
        for (int k = 0; k < V; ++k) {
          const double wk = which ? w[k] : d[k];
          s += wk;
          if (wk > 0.0) token = i + k;
          if (wk > 0.0 && s > border) break;
        }
        p.token[b] = token;
      }
      run += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (!found && lane == 0) {  // roundings put the border behind the warp's last token: the last one before it that can be drawn
      long long i = min(begin + (long long)per * round, (long long)p.vocab) - 1;
      for (; i > 0; --i) {
        const double q = minus ? (double)minus[i] : i == certain ? 1.0 : 0.0;
        if (usable(which ? (double)row[i] : (double)row[i] - q) > 0.0) break;
      }
      p.token[b] = max(i, 0ll);
    }
  }
  cluster_sync_all();  // nobody reads another's shared memory after this
}

}  // namespace

cudaError_t verify_drafts_launch(const VerifyDrafts& p, cudaStream_t stream) {
  auto fits = [](const float* t, long long seq, long long row) { return (uintptr_t)t % 16 == 0 && seq % 4 == 0 && row % 4 == 0; };
  const dim3 grid((unsigned)p.seqs * kVerifyCluster), block(kVerifyThreads);
  if (p.vocab % 4 == 0 && fits(p.target, p.target_seq, p.target_row) && (!p.draft || fits(p.draft, p.draft_seq, p.draft_row)))
    return launch_pdl(verify_drafts_kernel<4>, grid, block, 0, stream, 0, p);
  return launch_pdl(verify_drafts_kernel<1>, grid, block, 0, stream, 0, p);
}

}  // namespace dion
