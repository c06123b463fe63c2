// Drafted tokens against the target's probabilities: draft i stands while u_i q_i(x_i) < p_i(x_i); the token after the last
// that stands is drawn from max(p - q, 0) there (from p behind the last draft) by the inverse of the distribution.
#include <math.h>

#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"

namespace dion {

namespace {

constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ float usable(float w) { return w > 0.f && w < INFINITY ? w : 0.f; }

// One block per sequence.  Sums are in 64 bits, so that their order decides nothing: two orders differ by some 1e-16 of the
// whole, the border that a draw has to hit to tell them apart.
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyDrafts p) {
  __shared__ double sums[kVerifyThreads / 32 + 1];
  __shared__ int found;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long* tokens = p.tokens + b * p.tokens_seq;
  const float* u = p.uniforms + b * p.uniforms_seq;
  int a = 0;
  long long x = -1;
  for (; a < p.drafts; ++a) {
    x = tokens[a];
    if (x < 0 || x >= p.vocab) {
      if (threadIdx.x == 0) bad_argument(p.status);
      x = -1;
      break;
    }
    const double q = p.draft ? (double)p.draft[b * p.draft_seq + a * p.draft_row + x] : 1.0;
    if (!((double)u[a] * q < (double)p.target[b * p.target_seq + a * p.target_row + x])) break;
  }
  const bool all = a == p.drafts;
  const float* row = p.target + b * p.target_seq + a * p.target_row;
  const float* minus = p.draft && !all ? p.draft + b * p.draft_seq + a * p.draft_row : nullptr;
  auto weight = [&](int i, bool whole) -> double {
    const double w = row[i];
    double r = w;
    if (!whole) r = minus ? w - (double)minus[i] : i == x && !p.draft ? w - 1.0 : w;
    return r > 0.0 && r < INFINITY ? r : 0.0;
  };
  double total = 0.0, mine = 0.0, before = 0.0;
  const int per = (p.vocab + kVerifyThreads - 1) / kVerifyThreads, lo = min(threadIdx.x * per, p.vocab), hi = min(lo + per, p.vocab);
  bool whole = all;
  for (int round = 0; round < 2; ++round) {
    mine = 0.0;
    for (int i = lo; i < hi; ++i) mine += weight(i, whole);
    double s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double run = 0.0;
      for (int i = 0; i < kVerifyThreads / 32; ++i) {
        const double t = sums[i];
        sums[i] = run;
        run += t;
      }
      sums[kVerifyThreads / 32] = run;
      found = p.vocab - 1;
    }
    __syncthreads();
    total = sums[kVerifyThreads / 32];
    before = sums[warp] + s - mine;
    if (total > 0.0 || whole) break;
    whole = true;  // p - q leaves nothing: p itself
    __syncthreads();
  }
  const double border = (double)u[p.drafts] * total;
  double run = before;
  for (int i = lo; i < hi; ++i) {
    const double w = weight(i, whole);
    run += w;
    if (w > 0.0 && !(run <= border)) {
      atomicMin(&found, i);
      break;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.accepted[b] = a;
    p.token[b] = total > 0.0 ? found : 0;
  }
}

}  // namespace

cudaError_t verify_drafts_launch(const VerifyDrafts& p, cudaStream_t stream) {
  return launch_pdl(verify_drafts_kernel, dim3(p.seqs), dim3(kVerifyThreads), 0, stream, 0, p);
}

}  // namespace dion
