// Drafted tokens against the target's probabilities: draft i stands while u_i q_i(x_i) < p_i(x_i); the token after the last
// that stands is drawn from max(p - q, 0) there (from p behind the last draft) by the inverse of the distribution.
#include <math.h>

#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"
#include "umma.cuh"

namespace dion {

namespace {

constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 8;  // CTAs of a sequence
constexpr int kVerifyGroups = 64;  // parts of a warp's tokens that the search tells apart

// t - q in 64 bits where that is positive and finite, else zero
__device__ __forceinline__ double weight(float t, float q) {
  const double d = (double)t - (double)q;
  return t > q && d < INFINITY ? d : 0.0;
}

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
// CTA's sum over a warp's to one warp's tokens, which all warps of that CTA go through again, and to one group of these.
template <int V>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyDrafts p) {
  __shared__ double warp_sum[kVerifyWarps + 1], group_sum[kVerifyGroups];  // the warps' and the CTA's
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
  int certain = !p.draft && !all && x < p.vocab ? (int)x : -1;  // the draft's only token

  // V tokens of a lane from i on, all at once or none
  auto load = [&](const float* from, int i, float (&t)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) t[k] = 0.f;
    if (!from || i >= p.vocab) return;
    if constexpr (V == 4) {
      const float4 v = *reinterpret_cast<const float4*>(from + i);
      t[0] = v.x, t[1] = v.y, t[2] = v.z, t[3] = v.w;
    } else {
      t[0] = from[i];
    }
  };
  // tokens of this warp: `per` rounds of 32 * V
  constexpr int round = 32 * V, everybody = kVerifyCluster * kVerifyWarps * round;
  const int per = (int)(((long long)p.vocab + everybody - 1) / everybody);
  const int begin = (rank * kVerifyWarps + warp) * per * round;  // the bindings keep the vocabulary so far below 2^31
  // of rounds first .. last of the tokens from `from` on, in all lanes
  auto sum_of = [&](int from, int first, int last) {
    double sum = 0.0;
    constexpr int AHEAD = 16 / V;  // rounds whose loads are under way at once
    for (int r = first; r < last; r += AHEAD) {
      float t[AHEAD][V], q[AHEAD][V];
      const int i = from + r * round + lane * V;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        load(r + j < last ? row : nullptr, i + j * round, t[j]);
        load(r + j < last ? minus : nullptr, i + j * round, q[j]);
      }
      const int c = certain - i;
      if (certain >= 0 && c >= 0 && c < AHEAD * round) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (c == j * round + k) q[j][k] = 1.f;
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) sum += weight(t[j][k], q[j][k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };
  double total, before;
  for (;;) {
    const double sum = sum_of(begin, 0, per);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double s = 0.0;
      for (int i = 0; i < kVerifyWarps; ++i) s += warp_sum[i];
      warp_sum[kVerifyWarps] = s;
    }
    cluster_sync_all();
    const double mine = lane < kVerifyCluster ? remote(&warp_sum[kVerifyWarps], lane) : 0.0;
    total = before = 0.0;
    for (int i = 0; i < kVerifyCluster; ++i) {
      const double s = __shfl_sync(0xffffffffu, mine, i);
      if (i < rank) before += s;
      total += s;
    }
    if (total > 0.0 || (!minus && certain < 0)) break;
    minus = nullptr, certain = -1;  // p - q leaves nothing: p itself
    cluster_sync_all();
  }
  // The token is the first whose running sum exceeds the border.  The sums before a CTA are added up in one order by all of them, and
  // those before a warp's tokens and before a group of these by all warps of the CTA; each takes what lies before the next one's
  // start, the last one the rest, so that exactly one is searched, wherever roundings put the border.
  const double border = (double)u[p.drafts] * total;
  if (rank == 0 && threadIdx.x == 0) {
    p.accepted[b] = a;
    if (!(total > 0.0) || !(border < total)) p.token[b] = total > 0.0 && border >= total ? p.vocab - 1 : 0;  // the latter: a uniform that is none
  }
  if (total > 0.0 && border < total && (rank == 0 || before <= border) &&
      (rank == kVerifyCluster - 1 || before + warp_sum[kVerifyWarps] > border)) {
    int owner = 0;
    for (; owner < kVerifyWarps - 1 && before + warp_sum[owner] <= border; ++owner) before += warp_sum[owner];
    const int from = (rank * kVerifyWarps + owner) * per * round;
    const int each = (per + kVerifyGroups - 1) / kVerifyGroups, groups = (per + each - 1) / each;  // rounds of a group
    for (int g = warp; g < groups; g += kVerifyWarps) {
      const double sum = sum_of(from, g * each, min(per, (g + 1) * each));
      if (lane == 0) group_sum[g] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      int g = 0;
      for (; g < groups - 1 && before + group_sum[g] <= border; ++g) before += group_sum[g];
      bool found = false;
      for (int r = g * each; r < min(per, (g + 1) * each) && !found; ++r) {
        const int i = from + r * round + lane * V;
        float t[V], q[V];
        load(row, i, t);
        load(minus, i, q);
        double w[V], mine = 0.0;
#pragma unroll
        for (int k = 0; k < V; ++k) mine += w[k] = weight(t[k], i + k == certain ? 1.f : q[k]);
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && before + upto > border);
        found = over != 0;
        if (found && lane == __ffs(over) - 1) {
          double s = before + upto - mine;
          int token = i;
          for (int k = 0; k < V; ++k) {
            s += w[k];
            if (w[k] > 0.0) token = i + k;
            if (w[k] > 0.0 && s > border) break;
          }
          p.token[b] = token;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
      if (!found && lane == 0) {  // roundings put the border behind the group's last token: the last one that can be drawn up to there
        int i = min(from + min(per, (g + 1) * each) * round, p.vocab) - 1;
        while (i > 0 && !(weight(row[i], i == certain ? 1.f : minus ? minus[i] : 0.f) > 0.0)) --i;
        p.token[b] = max(i, 0);
      }
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
