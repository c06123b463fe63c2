// New tokens into the paged cache: rotation of queries and keys to their positions (with the norm over a head where the model
// has one), keys and values to their pages, queries to a tensor of their own.
//   y = (x1 c + x2 s, x2 c - x1 s),  y *= rsqrt(mean(y^2) + eps),   c, s: the tables' rows at lengths[b] + i
#include <cuda_bf16.h>

#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"

namespace dion {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int kAppendThreads = 256, kAppendTokens = 64;  // threads of a block, most tokens of one

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __bfloat1622float2(h[j]);
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 q;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
  return q;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(p), f);
  }
}

// HD / 16 lanes share a row (one head of one token): eight pairs each, 16 bytes from either half of the head.  A block takes
// `tokens_per_block` tokens, looks up their pages first and then goes through their H + 2 Hkv rows.
template <int HD, typename Table>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppend p) {
  constexpr int HALF = HD / 2, LPR = HD / 16;
  __shared__ long long k_at[kAppendTokens], v_at[kAppendTokens];  // of a token's rows in the pages; -1: it has none
  __shared__ int position[kAppendTokens];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * p.tokens_per_block, tokens = min(p.tokens_per_block, p.tokens - t0);
  if (blockIdx.x == 0) {  // offsets start at zero, never fall and end within the tokens
    bool bad = threadIdx.x == 0 && (p.offsets[0] != 0 || p.offsets[p.seqs] > p.tokens);
    for (int b = threadIdx.x; b < p.seqs; b += kAppendThreads) bad |= p.offsets[b] > p.offsets[b + 1];
    if (bad) bad_argument(p.status);
  }
  for (int i = warp; i < tokens; i += kAppendThreads / 32) {
    const int row = t0 + i, b = sequence_of(p.offsets, p.seqs, row, lane);
    if (lane == 0) {
      const int first = p.offsets[b], end = p.offsets[b + 1];
      long long ka = -1, va = -1;
      int pos = 0;
      if (row >= first && row < end) {
        const long long at = (long long)p.lengths[b] + ((long long)row - first), slot = at >> p.page_shift;
        int page = -1;
        if (p.lengths[b] >= 0 && at < p.table_rows && slot < p.max_pages) page = p.page_table[(long long)b * p.table_pitch + slot];
        if (page >= 0 && page < p.pages) {
          const int in_page = (int)(at & ((1 << p.page_shift) - 1));
          ka = page * p.k_page + in_page * p.k_row;
          va = page * p.v_page + in_page * p.v_row;
          pos = (int)at;
        } else {
          bad_argument(p.status);
        }
      }
      k_at[i] = ka, v_at[i] = va, position[i] = pos;
    }
  }
  __syncthreads();
  const int rows = p.heads + 2 * p.kv_heads, units = rows * LPR;
  const int total = (tokens * units + 31) / 32 * 32;  // whole warps, for the shuffles
  for (int u = threadIdx.x; u < total; u += kAppendThreads) {
    const bool live = u < tokens * units;
    const int i = live ? u / units : 0, r = live ? (u - i * units) / LPR : 0, col = (u % LPR) * 8;
    const long long token = t0 + i;
    const long long to_k = k_at[i];
    const bf16* src;
    bf16* dst;
    if (r < p.heads) {
      src = p.q + token * p.q_token + r * p.q_head;
      dst = p.q_out + (token * p.heads + r) * HD;
    } else if (r < p.heads + p.kv_heads) {
      const int h = r - p.heads;
      src = p.k + token * p.k_token + h * p.k_in_head;
      dst = p.k_pages + to_k + h * p.k_head;
    } else {
      const int h = r - p.heads - p.kv_heads;
      src = p.v + token * p.v_token + h * p.v_in_head;
      dst = p.v_pages + v_at[i] + h * p.v_head;
    }
    uint4 a = *reinterpret_cast<const uint4*>(src + col), b = *reinterpret_cast<const uint4*>(src + col + HALF);
    const bool turn = r < p.heads + p.kv_heads;
    float x1[8], x2[8], c[8], s[8], y1[8], y2[8], ss = 0.f;
    unpack8(a, x1);
    unpack8(b, x2);
    const long long at = (long long)position[i] * p.cos_row + col, sat = (long long)position[i] * p.sin_row + col;
    load8(reinterpret_cast<const Table*>(p.cos) + at, c);
    load8(reinterpret_cast<const Table*>(p.sin) + sat, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y1[j] = x1[j] * c[j] + x2[j] * s[j];
      y2[j] = x2[j] * c[j] - x1[j] * s[j];
      ss += y1[j] * y1[j] + y2[j] * y2[j];
    }
    if (p.eps >= 0.f) {
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float f = rsqrtf(ss / (float)HD + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y1[j] *= f, y2[j] *= f;
    }
    if (turn) a = pack8(y1), b = pack8(y2);
    if (to_k < 0) {  // nobody's row: its query becomes zero, nothing goes to the pages
      a = b = make_uint4(0, 0, 0, 0);
      if (r >= p.heads) continue;
    }
    if (live) {
      *reinterpret_cast<uint4*>(dst + col) = a;
      *reinterpret_cast<uint4*>(dst + col + HALF) = b;
    }
  }
}

}  // namespace

cudaError_t paged_append_launch(PagedAppend p, int head_dim, bool wide_tables, cudaStream_t stream) {
  if (p.tokens <= 0) return cudaSuccess;
  const int units = (p.heads + 2 * p.kv_heads) * (head_dim / 16);
  // two rounds of a block's threads
  p.tokens_per_block = units >= 2 * kAppendThreads ? 1 : 2 * kAppendThreads / units;
  if (p.tokens_per_block > kAppendTokens) p.tokens_per_block = kAppendTokens;
  const dim3 grid((p.tokens + p.tokens_per_block - 1) / p.tokens_per_block), block(kAppendThreads);
  if (head_dim == 64)
    return wide_tables ? launch_pdl(paged_append_kernel<64, float>, grid, block, 0, stream, 0, p)
                       : launch_pdl(paged_append_kernel<64, bf16>, grid, block, 0, stream, 0, p);
  if (head_dim == 128)
    return wide_tables ? launch_pdl(paged_append_kernel<128, float>, grid, block, 0, stream, 0, p)
                       : launch_pdl(paged_append_kernel<128, bf16>, grid, block, 0, stream, 0, p);
  return cudaErrorInvalidValue;
}

}  // namespace dion
