// Causal attention of new tokens over a paged cache of keys and values:
//   out = softmax(scale q K[0..p]^T) V[0..p],   p = lengths[b] + i of row i of sequence b.
#include <cuda_bf16.h>
#include <math.h>

#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"

namespace dion {

namespace {

typedef __nv_bfloat16 bf16;

// One warp per query row: its lanes share the head dimension, keys one after the other with the running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttention p) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (blockIdx.x == 0) {
    bool bad = threadIdx.x == 0 && (p.offsets[0] != 0 || p.offsets[p.seqs] > p.tokens);
    for (int b = threadIdx.x; b < p.seqs; b += 128) bad |= p.offsets[b] > p.offsets[b + 1];
    if (bad) bad_argument(p.status);
  }
  if (w >= (long long)p.tokens * p.heads) return;
  const int row = (int)(w / p.heads), h = (int)(w - (long long)row * p.heads), hk = h / (p.heads / p.kv_heads);
  const int b = sequence_of(p.offsets, p.seqs, row, lane);
  const int first = p.offsets[b], end = p.offsets[b + 1];
  long long keys = 0;
  if (row >= first && row < end) {
    const long long most = (long long)p.max_pages << p.page_shift;
    keys = (long long)p.lengths[b] + ((long long)row - first) + 1;
    if (p.lengths[b] < 0 || keys > most || (long long)end - first > p.max_new) {
      bad_argument(p.status);
      keys = 0;
    }
  }
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = __bfloat162float(p.q[row * p.q_token + h * p.q_head + lane * E + i]) * p.scale * 1.4426950408889634f;
    o[i] = 0.f;
  }
  for (long long j = 0; j < keys; ++j) {
    const int page = p.page_table[(long long)b * p.table_pitch + (j >> p.page_shift)];
    if (page < 0 || page >= p.pages) {
      bad_argument(p.status);
      continue;
    }
    const int at = (int)(j & ((1 << p.page_shift) - 1));
    const bf16* k = p.k_pages + page * p.k_page + at * p.k_row + hk * p.k_head + lane * E;
    const bf16* v = p.v_pages + page * p.v_page + at * p.v_row + hk * p.v_head + lane * E;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += q[i] * __bfloat162float(k[i]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float m2 = fmaxf(m, s), a = m2 == -INFINITY ? 1.f : exp2f(m - m2), e = m2 == -INFINITY ? 0.f : exp2f(s - m2);
    l = l * a + e;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * a + e * __bfloat162float(v[i]);
    m = m2;
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    p.out[((long long)row * p.heads + h) * D + lane * E + i] = __float2bfloat16(l > 0.f ? o[i] / l : 0.f);
}

}  // namespace

cudaError_t paged_attention_launch(const PagedAttention& p, int head_dim, cudaStream_t stream) {
  const long long warps = (long long)p.tokens * p.heads;
  const dim3 grid((unsigned)((warps + 3) / 4));
  if (head_dim == 64) return launch_pdl(paged_attention_kernel<64>, grid, dim3(128), 0, stream, 0, p);
  if (head_dim == 128) return launch_pdl(paged_attention_kernel<128>, grid, dim3(128), 0, stream, 0, p);
  return cudaErrorInvalidValue;
}

}  // namespace dion
