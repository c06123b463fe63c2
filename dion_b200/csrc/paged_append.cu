// New tokens into the paged cache: rotation of queries and keys to their positions (with the norm over a head where the model
// has one), keys and values to their pages, queries to a tensor of their own.
//   y = (x1 c + x2 s, x2 c - x1 s),  y *= rsqrt(mean(y^2) + eps),   c, s: the tables' rows at lengths[b] + i
#include <cuda_bf16.h>

#include "attention.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"

namespace dion {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int kAppendThreads = 256;  // of a block, at most
// Tokens of a block, where there are many.  16384 tokens, 32 heads and 8 kv heads of 128 (us): 68 with 2, 68.5 with 4, 94 with 8;
// 33 prompts of up to 900, 12 heads of 64, with the norm: 32, 33, 44
constexpr int kAppendTokens = 2;

// eight values as four pairs of fp32
__device__ __forceinline__ void unpack8(const uint4& q, f32x2 (&f)[4]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack8(const f32x2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    unpack2(f[j], a, b);
    w[j] = pack_bf16x2(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, f32x2 (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = pack2(a.x, a.y), f[1] = pack2(a.z, a.w), f[2] = pack2(b.x, b.y), f[3] = pack2(b.z, b.w);
  } else {
    unpack8(*reinterpret_cast<const uint4*>(p), f);
  }
}

// HD / 16 lanes share a row (one head of one token): eight pairs each, 16 bytes from either half of the head.  A block takes T tokens
// and as many of their rows as it has threads for, every thread the same row of each token, so that its addresses move on by one
// stride.  Bound by memory: all loads of a thread are under way before it looks up where the rows go, and two fp32 operations go in one
// instruction, as with single ones the issue slots were half full.  Six blocks of 256 threads an SM: 67 and 30 us for
// the cases at kAppendTokens, 72 and 33 with the registers that the compiler would take.
template <int HD, int T, typename Table>
__global__ void __launch_bounds__(kAppendThreads, T == 1 ? 1 : 6) paged_append_kernel(const PagedAppend p) {
  constexpr int HALF = HD / 2, LPR = HD / 16;
  __shared__ long long k_at[T], v_at[T];  // of a token's rows in the pages; -1: it has none
  __shared__ int position[T];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, col = (threadIdx.x % LPR) * 8;
  const int t0 = (int)blockIdx.x * T, r = (int)(blockIdx.y * (blockDim.x / LPR) + threadIdx.x / LPR);
  const bool of_q = r < p.heads, of_k = !of_q && r < p.heads + p.kv_heads, there = r < p.heads + 2 * p.kv_heads;
  const int h = of_q ? r : of_k ? r - p.heads : r - p.heads - p.kv_heads;
  uint4 lo[T], hi[T];
  if (there) {
    const long long step = of_q ? p.q_token : of_k ? p.k_token : p.v_token;
    const bf16* src = (of_q ? p.q : of_k ? p.k : p.v) + t0 * step + h * (of_q ? p.q_head : of_k ? p.k_in_head : p.v_in_head) + col;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      if (T == 1 || t0 + j < p.tokens) {
        lo[j] = *reinterpret_cast<const uint4*>(src);
        hi[j] = *reinterpret_cast<const uint4*>(src + HALF);
      }
      src += step;
    }
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) {  // offsets start at zero, never fall and end within the tokens
    bool bad = threadIdx.x == 0 && (p.offsets[0] != 0 || p.offsets[p.seqs] > p.tokens);
    for (int b = threadIdx.x; b < p.seqs; b += blockDim.x) bad |= p.offsets[b] > p.offsets[b + 1];
    if (bad) bad_argument(p.status);
  }
  for (int j = threadIdx.x / 32; j < T; j += blockDim.x / 32) {  // a warp per token
    const int row = t0 + j, b = sequence_of(p.offsets, p.seqs, row, lane);
    if (lane == 0) {
      const int first = p.offsets[b], end = p.offsets[b + 1];
      long long ka = -1, va = -1;
      int pos = 0;
      if (row >= first && row < end && row < p.tokens) {
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
      k_at[j] = ka, v_at[j] = va, position[j] = pos;
    }
  }
  __syncthreads();
  if (!there) return;
  const unsigned row_lanes = ((1u << LPR) - 1) << (lane & ~(LPR - 1));  // the lanes of this row: all or none of them get here
  bf16* to = (of_q ? p.q_out + ((long long)t0 * p.heads + h) * HD : of_k ? p.k_pages + h * p.k_head : p.v_pages + h * p.v_head) + col;
#pragma unroll
  for (int j = 0; j < T; ++j) {
    if (T > 1 && t0 + j >= p.tokens) break;
    const long long at = of_k ? k_at[j] : v_at[j];
    uint4 a = lo[j], b = hi[j];
    if ((of_q || of_k) && at >= 0) {  // nobody's row has no position, and the tables may not have a row either
      f32x2 x1[4], x2[4], c[4], s[4];
      unpack8(a, x1);
      unpack8(b, x2);
      load8(reinterpret_cast<const Table*>(p.cos) + (long long)position[j] * p.cos_row + col, c);
      load8(reinterpret_cast<const Table*>(p.sin) + (long long)position[j] * p.sin_row + col, s);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the operations of the training kernels in their order, and so their bits
        const f32x2 minus_s = s[e] ^ 0x8000000080000000ull;
        const f32x2 y1 = fma2(x1[e], c[e], mul2(x2[e], s[e])), y2 = fma2(x2[e], c[e], mul2(x1[e], minus_s));
        x1[e] = y1, x2[e] = y2;
        float s0, s1;
        unpack2(fma2(y1, y1, mul2(y2, y2)), s0, s1);
        ss += s0;
        ss += s1;
      }
      if (p.eps >= 0.f) {
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(row_lanes, ss, o);
        const float f = rsqrtf(ss / (float)HD + p.eps);
        const f32x2 f2 = pack2(f, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) x1[e] = mul2(x1[e], f2), x2[e] = mul2(x2[e], f2);
      }
      a = pack8(x1);
      b = pack8(x2);
    }
    if (at < 0) a = b = make_uint4(0, 0, 0, 0);  // nobody's row: its query becomes zero, nothing goes to the pages
    if (of_q || at >= 0) {
      bf16* dst = of_q ? to + (long long)j * p.heads * HD : to + at;
      *reinterpret_cast<uint4*>(dst) = a;
      *reinterpret_cast<uint4*>(dst + HALF) = b;
    }
  }
}

template <int HD, typename Table>
cudaError_t append_launch(const PagedAppend& p, cudaStream_t stream) {
  constexpr int step = 32 / (HD / 16);  // rows of a warp
  const int rows = p.heads + 2 * p.kv_heads, most = kAppendThreads / 32 * step;
  const int parts = (rows + most - 1) / most, each = ((rows + parts - 1) / parts + step - 1) / step * step;  // blocks of a token, rows of one
  if (parts > 65535) return cudaErrorInvalidValue;
  const dim3 block(each * (HD / 16));
  // One token a block up to eight blocks per SM, where the shorter chain counts.  In a graph (us, one token / kAppendTokens): 6 + 2 x 6
  // heads of 128, 64 tokens 2.4 / 2.9, 900 3.3 / 4.4, 1200 5.1 / 5.4, 2400 8.5 / 7.6; 32 + 2 x 8 (two blocks a token), 450 tokens
  // 5.5 / 6.0, 600 6.8 / 6.5, 9600 51.4 / 44.4; 12 + 2 x 12 of 64, 900 3.3 / 4.3, 2400 8.5 / 7.2.
  if ((long long)p.tokens * parts <= 8ll * attn_grid(1 << 20))
    return launch_pdl(paged_append_kernel<HD, 1, Table>, dim3(p.tokens, parts), block, 0, stream, 0, p);
  return launch_pdl(paged_append_kernel<HD, kAppendTokens, Table>, dim3((p.tokens + kAppendTokens - 1) / kAppendTokens, parts), block, 0, stream, 0, p);
}

}  // namespace

cudaError_t paged_append_launch(const PagedAppend& p, int head_dim, bool wide_tables, cudaStream_t stream) {
  if (p.tokens <= 0) return cudaSuccess;
  if (head_dim == 64) return wide_tables ? append_launch<64, float>(p, stream) : append_launch<64, bf16>(p, stream);
  if (head_dim == 128) return wide_tables ? append_launch<128, float>(p, stream) : append_launch<128, bf16>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace dion
