// Causal attention of new tokens over a paged cache of keys and values:
//   out = softmax(scale q K[0..p]^T) V[0..p],   p = lengths[b] + i of row i of sequence b.
//
// The rows of a sequence that share a kv head (new tokens x heads of its group, token by token) make one tile of queries.  The keys
// are taken once per tile with the running maximum and sum of a softmax, and all keys of all tiles are dealt out evenly over the
// CTAs, whatever the lengths: a CTA's share may end inside a tile, whose parts a second kernel then joins.  The shares follow from
// the sizes alone, so a call gives the same bits every time.
#include <cuda.h>
#include <cuda_bf16.h>
#include <math.h>

#include <atomic>

#include "attention.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "pdl.cuh"
#include "per_device.h"
#include "umma.cuh"

namespace dion {

namespace {

typedef __nv_bfloat16 bf16;

// ---------------------------------------------------------------------------------- the work and its shares

// A sequence of the call: rows first .. first + n, keys = cached + new.  n = 0 where there is nothing to do or something is wrong.
struct Sequence {
  int first, n, keys;
  bool bad;
};
__device__ __forceinline__ Sequence sequence(const PagedAttention& p, int b) {
  const long long first = p.offsets[b], end = p.offsets[b + 1], cached = p.lengths[b], n = end - first;
  Sequence s{0, 0, 0, false};
  if (n == 0) return s;
  const long long most = min((long long)p.max_pages << p.page_shift, 0x7fffffffll - 1024);
  s.bad = first < 0 || n < 0 || end > p.tokens || cached < 0 || cached + n > most || n > p.max_new;
  if (!s.bad) s = Sequence{(int)first, (int)n, (int)(cached + n), false};
  return s;
}

// ---------------------------------------------------------------------------------- few rows per kv head: mma.sync

constexpr int kKeys = 64;               // keys of a stage
constexpr int kRowsThreads = 32 * 5;    // four warps of products and one that loads
constexpr int kShareUnits = 2;          // stages that are worth a CTA

template <int D_, int WM_>
struct Rows {
  static constexpr int D = D_, WM = WM_, WK = 4 / WM, TR = 16 * WM;  // warps along the rows and along the keys, rows of a tile
  static constexpr int PANELS = D / 64, PANEL = kKeys * 128, STAGE = 2 * PANELS * PANEL;  // bytes; K panels, then V panels
  static constexpr int STAGES = D == 128 ? 3 : 6;
  static constexpr int EXCHANGE = WK > 1 ? 2 * 16 * D * 4 : 0;  // accumulators of two warps on their way to their neighbours
  static constexpr int SMEM = STAGES * STAGE + EXCHANGE + 1024;
  static_assert(SMEM <= 115712, "two CTAs per SM");
};

// What a CTA leaves for the join.  Slot 2c holds its first tile where an earlier CTA has begun it, slot 2c + 1 its last one where a
// later CTA ends it.
struct Share {
  int b, kv_head;   // of the tile in slot 2c + 1; b = -1: none
  int continues;    // slot 2c is filled
  int ends;         // ... and its tile ends here
};
struct Parts {
  float* acc;    // [slot][rows of a tile][head_dim], not normalised
  float2* ml;    // [slot][rows of a tile]: maximum (log2 units) and sum
  Share* share;  // per CTA
  int rows;      // of a tile
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk `chunk` of a 128-byte row in the 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ void products_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the four warps of products

// Where a CTA's share stands: kv head `head` of sequence b, from stage `unit` on, `left` stages to go.
struct Walk {
  int b, head, unit, units;
  long long left;
  Sequence s;
};
template <int TR>
__device__ __forceinline__ int units_of(const PagedAttention& p, const Sequence& s) {
  return (long long)s.n * (p.heads / p.kv_heads) <= TR ? (s.keys + kKeys - 1) / kKeys : 0;
}
template <int TR>
__device__ __forceinline__ void next_tile(Walk& w, const PagedAttention& p, int done) {
  w.left -= done;
  w.unit = 0;
  if (++w.head < p.kv_heads) return;
  w.head = 0;
  w.units = 0;
  while (w.left > 0 && w.units == 0 && ++w.b < p.seqs) {
    w.s = sequence(p, w.b);
    w.units = units_of<TR>(p, w.s);
  }
}

// This CTA's share of all stages of all tiles, found by the whole block.  sums: a value per thread of the block and one more.
template <int TR>
__device__ Walk my_share(const PagedAttention& p, long long* sums, long long* found) {
  const int per = (p.seqs + kRowsThreads - 1) / kRowsThreads, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int lo = min(t * per, p.seqs), hi = min(lo + per, p.seqs);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += (long long)units_of<TR>(p, sequence(p, b)) * p.kv_heads;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[warp] = upto;
  if (t == 0) found[0] = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < kRowsThreads / 32; ++i) {
    if (i < warp) upto += sums[i];
    total += sums[i];
  }
  const long long ctas = min((long long)gridDim.x, (total + kShareUnits - 1) / kShareUnits);
  long long from = 0, to = 0;
  if (blockIdx.x < ctas) from = total * blockIdx.x / ctas, to = total * (blockIdx.x + 1) / ctas;
  if (from < to && upto - mine <= from && from < upto) {  // the thread whose sequences hold the start
    long long at = upto - mine;
    for (int b = lo; b < hi; ++b) {
      const long long u = (long long)units_of<TR>(p, sequence(p, b)) * p.kv_heads;
      if (from < at + u) {
        found[0] = b;
        found[1] = from - at;
        break;
      }
      at += u;
    }
  }
  __syncthreads();
  Walk w{(int)found[0], 0, 0, 0, to - from, {}};
  if (w.b < 0) w.left = 0;
  if (w.left > 0) {
    w.s = sequence(p, w.b);
    w.units = units_of<TR>(p, w.s);
    w.head = (int)(found[1] / w.units);
    w.unit = (int)(found[1] - (long long)w.head * w.units);
  }
  return w;
}

// Bound by the bandwidth of the cache: 64 keys are 32 KB (head dimension 128), which an SM gets in 1400 cycles, and take four
// warps some 600.  So the legacy products, whose tiles are 16 rows high, do: the rows of single tokens fill no more.  A warp loads
// 64 keys a stage by TMA, the boxes of several pages where they are smaller; where the rows fit one 16-row tile the four others
// take 16 keys each and join their sums per tile, else they share the keys and have rows of their own.
template <typename C>
__global__ void __launch_bounds__(kRowsThreads, 2)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const PagedAttention p,
                  const Parts parts, const FastDiv by_group) {
  constexpr int D = C::D, WK = C::WK, TR = C::TR;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* exchange = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE + C::EXCHANGE);
  uint64_t* empty = full + C::STAGES;
  long long* sums = reinterpret_cast<long long*>(empty + C::STAGES);
  long long* found = sums + kRowsThreads / 32;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(found + 2);
  float2* stats = reinterpret_cast<float2*>(found + 3);  // [warp][16 rows]
  const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {  // the 128-byte swizzle repeats every 1024 bytes
    if (threadIdx.x == 0) {
      bad_argument(p.status);
      parts.share[blockIdx.x] = Share{-1, 0, 0, 0};
    }
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  pdl_trigger();
  pdl_wait();
  Walk w = my_share<TR>(p, sums, found);
  const int group = p.heads / p.kv_heads;
  Ring<C::STAGES> ring;

  if (warp == 4) {
    // ------------------------------------------------------------------ loads
    const int shift = p.page_shift, box = min(kKeys, 1 << shift), boxes = kKeys / box;
    while (w.left > 0) {
      const int end = (int)min((long long)w.units, w.unit + w.left);
      const int* table = p.page_table + (long long)w.b * p.table_pitch;
      const int used = (int)(((long long)w.s.keys + (1 << shift) - 1) >> shift);
      int held = 0, have = 0, page = 0;  // lane i: page held + i, for i < have
      for (int u = w.unit; u < end; ++u) {
        const int key = u * kKeys, first = key >> shift, count = min(boxes, used - first);
        if (first < held || first + count > held + have) {
          held = first;
          have = min(32, used - first);
          if (lane < have) {
            page = table[first + lane];
            if (page < 0 || page >= p.pages) {
              bad_argument(p.status);
              page = 0;
            }
          }
        }
        const int mine = __shfl_sync(0xffffffffu, page, (first - held + lane) & 31);
        if (!mbar_wait(&empty[ring.s], ring.ph ^ 1u, abort_flag)) {
          *abort_flag = 1;
          if (lane == 0) atomicCAS(p.status, 0, kStatusProducerTimeout);
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        uint8_t* stage = smem + ring.s * C::STAGE;
        if (lane == 0) mbar_arrive_expect_tx(&full[ring.s], count * box * (4 * D));
        __syncwarp();
        if (lane < count) {
          const int at = key & ((1 << shift) - 1);  // inside a page larger than a stage
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c) {
            tma_load_4d(stage + c * C::PANEL + lane * box * 128, &tmap_k, &full[ring.s], c * 64, w.head, at, mine);
            tma_load_4d(stage + (C::PANELS + c) * C::PANEL + lane * box * 128, &tmap_v, &full[ring.s], c * 64, w.head, at, mine);
          }
        }
        ring.next();
      }
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
      next_tile<TR>(w, p, end - w.unit);
    }
  } else {
    // ------------------------------------------------------------------ products
    // A wait that gives up raises the abort flag and the warp goes on without waiting, so that the barriers of the four are met.
    const int wm = warp % C::WM, wk = warp / C::WM;
    constexpr int KG = kKeys / WK / 16;  // groups of 16 keys that this warp has in a stage
    const int key0 = wk * (kKeys / WK), quad = lane >> 2, pair = (lane & 3) * 2;
    const float scale = p.scale * 1.4426950408889634f;
    bool dead = false;
    Share share{-1, 0, 0, 0};
    bool first_tile = true;
    while (w.left > 0) {
      const int begin = w.unit, end = (int)min((long long)w.units, w.unit + w.left), rows = w.s.n * group;
      const int cached = w.s.keys - w.s.n;
      // queries of rows quad and quad + 8, and how many keys these see
      uint32_t q[D / 16][4];
      int sees[2];
      long long to[2];  // their rows of the result
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = wm * 16 + quad + 8 * i, token = by_group(min(r, rows - 1)), h = w.head * group + (min(r, rows - 1) - token * group);
        const bf16* src = p.q + (w.s.first + token) * p.q_token + h * p.q_head + pair;
        sees[i] = cached + token + 1;
        to[i] = r < rows ? ((long long)(w.s.first + token) * p.heads + h) * D : -1;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          q[kk][i] = *reinterpret_cast<const uint32_t*>(src + kk * 16);
          q[kk][2 + i] = *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8);
        }
      }
      float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      for (int u = begin; u < end; ++u) {
        if (!dead && !mbar_wait(&full[ring.s], ring.ph, abort_flag)) {
          *abort_flag = 1;
          atomicCAS(p.status, 0, kStatusMmaTimeout);
        }
        dead = __any_sync(0xffffffffu, *abort_flag != 0);
        const uint32_t ks = smem_u32(smem) + ring.s * C::STAGE, vs = ks + C::PANELS * C::PANEL;
        const int at = u * kKeys + key0;  // the first key of this warp
        float s[2 * KG][4];
#pragma unroll
        for (int i = 0; i < 2 * KG; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int g = 0; g < KG; ++g) {
            uint32_t k[4];
            const uint32_t row = key0 + g * 16 + (lane & 7) + ((lane & 16) >> 1), chunk = (kk & 3) * 2 + ((lane >> 3) & 1);
            ldmatrix4(ks + (kk >> 2) * C::PANEL + swizzled(row, chunk), k);
            mma16816(s[2 * g], q[kk], k[0], k[1]);
            mma16816(s[2 * g + 1], q[kk], k[2], k[3]);
          }
        if (at + KG * 16 > cached + 1) {  // beyond what the first token sees
#pragma unroll
          for (int i = 0; i < 2 * KG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (at + i * 8 + pair + (j & 1) >= sees[j >> 1]) s[i][j] = -INFINITY;
        }
        float mx[2] = {-INFINITY, -INFINITY}, f[2], neg[2];
#pragma unroll
        for (int i = 0; i < 2 * KG; ++i) {
          mx[0] = fmaxf(mx[0], fmaxf(s[i][0], s[i][1]));
          mx[1] = fmaxf(mx[1], fmaxf(s[i][2], s[i][3]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float m2 = fmaxf(m[i], quad_max(mx[i]) * scale);
          neg[i] = m2 == -INFINITY ? 0.f : -m2;  // nothing seen yet
          f[i] = fast_exp2(m[i] + neg[i]);
          m[i] = m2;
          l[i] *= f[i];
        }
        uint32_t pr[2 * KG][2];  // weights in bf16, as the products take them; their sum is that of the unrounded ones
#pragma unroll
        for (int i = 0; i < 2 * KG; ++i) {
          const float e0 = fast_exp2(fmaf(s[i][0], scale, neg[0])), e1 = fast_exp2(fmaf(s[i][1], scale, neg[0]));
          const float e2 = fast_exp2(fmaf(s[i][2], scale, neg[1])), e3 = fast_exp2(fmaf(s[i][3], scale, neg[1]));
          l[0] += e0 + e1;
          l[1] += e2 + e3;
          pr[i][0] = pack_bf16x2(e0, e1);
          pr[i][1] = pack_bf16x2(e2, e3);
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) o[i][0] *= f[0], o[i][1] *= f[0], o[i][2] *= f[1], o[i][3] *= f[1];
        }
        const bool ragged = at + KG * 16 > w.s.keys;  // what lies behind the last key may be no numbers: taken as zeros
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const uint32_t a[4] = {pr[2 * g][0], pr[2 * g][1], pr[2 * g + 1][0], pr[2 * g + 1][1]};
          const int left = w.s.keys - (at + g * 16) - pair;  // of the keys from this lane's first on
          const uint32_t keep0 = (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u);
          const uint32_t keep1 = (left > 8 ? 0xffffu : 0u) | (left > 9 ? 0xffff0000u : 0u);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t v[4];
            const uint32_t row = key0 + g * 16 + (lane & 15), chunk = (c & 3) * 2 + (lane >> 4);
            ldmatrix4_trans(vs + (c >> 2) * C::PANEL + swizzled(row, chunk), v);
            if (ragged) v[0] &= keep0, v[1] &= keep1, v[2] &= keep0, v[3] &= keep1;
            mma16816(o[2 * c], a, v[0], v[1]);
            mma16816(o[2 * c + 1], a, v[2], v[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ring.s]);
        ring.next();
      }
      l[0] = quad_sum(l[0]);
      l[1] = quad_sum(l[1]);
      if constexpr (WK > 1) {
        // the warps that had the same rows join their sums
        if ((lane & 3) == 0) {
          stats[warp * 16 + quad] = make_float2(m[0], l[0]);
          stats[warp * 16 + quad + 8] = make_float2(m[1], l[1]);
        }
        products_sync();
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int k = 0; k < WK; ++k) top = fmaxf(top, stats[(wm + k * C::WM) * 16 + quad + 8 * i].x);
          const float neg = top == -INFINITY ? 0.f : -top;
#pragma unroll
          for (int k = 0; k < WK; ++k) {
            const float2 t = stats[(wm + k * C::WM) * 16 + quad + 8 * i];
            sum += t.y * fast_exp2(t.x + neg);
          }
          f[i] = fast_exp2(m[i] + neg);
          m[i] = top;
          l[i] = sum;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] *= f[0], o[i][1] *= f[0], o[i][2] *= f[1], o[i][3] *= f[1];
#pragma unroll
        for (int step = 2; step > 0; step >>= 1) {  // warps step .. 2 step hand theirs to the ones before
          if (step < C::WM) break;
          if (warp >= step && warp < 2 * step) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
              *reinterpret_cast<float4*>(exchange + (((warp - step) * (D / 8) + i) * 32 + lane) * 4) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
          }
          products_sync();
          if (warp < step) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              const float4 t = *reinterpret_cast<const float4*>(exchange + ((warp * (D / 8) + i) * 32 + lane) * 4);
              o[i][0] += t.x, o[i][1] += t.y, o[i][2] += t.z, o[i][3] += t.w;
            }
          }
          products_sync();
        }
      }
      const bool starts = begin == 0, ends = end == w.units;
      if (wk == 0) {
        if (starts && ends) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (to[i] < 0) continue;
            const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<uint32_t*>(p.out + to[i] + c * 8 + pair) = pack_bf16x2(o[c][2 * i] * inv, o[c][2 * i + 1] * inv);
          }
        } else {
          const long long slot = 2 * (long long)blockIdx.x + (starts ? 1 : 0);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (to[i] < 0) continue;
            const long long r = slot * TR + wm * 16 + quad + 8 * i;
            if ((lane & 3) == 0) parts.ml[r] = make_float2(m[i], l[i]);
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<float2*>(parts.acc + r * D + c * 8 + pair) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
          }
        }
      }
      if (starts && !ends) share.b = w.b, share.kv_head = w.head;
      if (!starts && first_tile) share.continues = 1, share.ends = ends;
      first_tile = false;
      next_tile<TR>(w, p, end - begin);
    }
    if (threadIdx.x == 0) parts.share[blockIdx.x] = share;
  }
  __syncthreads();
  if (*abort_flag != 0) {
    // a wait gave up: let copies that are still in flight land before the CTA retires
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
}

// Joins the parts of tiles that several CTAs had, writes zeros to rows that are nobody's and reports what is wrong with the
// sequences.  Block (c, y) has the tile that CTA c began, rows y, y + 8 * gridDim.y ..., one per warp.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttention p, const Parts parts, int ctas) {
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;
  const int group = p.heads / p.kv_heads;
  if (blockIdx.y == 0) {  // sequences c, c + gridDim.x ... and a share of the rows behind the last
    auto clear = [&](long long lo, long long hi) {
      lo = max(lo, 0ll);
      hi = min(hi, (long long)p.tokens);
      const long long per_row = (long long)p.heads * D / 8;
      for (long long i = lo * per_row + threadIdx.x; i < hi * per_row; i += 256) reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
    };
    for (int b = c; b < p.seqs; b += gridDim.x) {
      if (sequence(p, b).bad) {
        if (threadIdx.x == 0) bad_argument(p.status);
        clear(p.offsets[b], p.offsets[b + 1]);
      }
    }
    if (c == 0 && threadIdx.x == 0 && p.offsets[0] != 0) bad_argument(p.status);
    for (long long r = (long long)p.offsets[p.seqs] + c; r < p.tokens; r += gridDim.x) clear(r, r + 1);
  }
  if (c >= ctas) return;
  const Share mine = parts.share[c];
  if (mine.b < 0) return;
  const Sequence s = sequence(p, mine.b);
  int last = c;  // the CTA that ends the tile
  for (bool more = true; more;) {
    const int i = last + 1 + lane;
    const bool stop = i >= ctas || !parts.share[i].continues || parts.share[i].ends;
    const unsigned at = __ballot_sync(0xffffffffu, stop);
    more = at == 0;
    last += more ? 32 : __ffs(at);
  }
  last = min(last, ctas - 1);
  constexpr int E = D / 32;
  for (int r = blockIdx.y * 8 + warp; r < s.n * group; r += 8 * gridDim.y) {
    float top = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int base = c; base <= last; base += 32) {
      const int i = base + lane;
      const long long slot = i == c ? 2ll * c + 1 : 2ll * i;
      const float2 t = i <= last ? parts.ml[slot * parts.rows + r] : make_float2(-INFINITY, 0.f);
      float most = t.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float top2 = fmaxf(top, most), neg = top2 == -INFINITY ? 0.f : -top2, f = fast_exp2(top + neg), mw = fast_exp2(t.x + neg);
      float part = t.y * mw;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      sum = sum * f + part;
      top = top2;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
      const int n = min(32, last + 1 - base);
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float wk = __shfl_sync(0xffffffffu, mw, k);
        const long long from = (base + k == c ? 2ll * c + 1 : 2ll * (base + k)) * parts.rows + r;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += wk * parts.acc[from * D + e * 32 + lane];
      }
    }
    const int token = r / group, h = mine.kv_head * group + (r - token * group);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      p.out[((long long)(s.first + token) * p.heads + h) * D + e * 32 + lane] = __float2bfloat16(acc[e] * inv);
  }
}

// ---------------------------------------------------------------------------------- many rows

// The sequences whose rows are too many for the kernel above.  One warp per query row: its lanes share the head dimension, keys one after the other with the running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttention p, int above) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)p.tokens * p.heads) return;
  const int row = (int)(w / p.heads), h = (int)(w - (long long)row * p.heads), hk = h / (p.heads / p.kv_heads);
  const int b = sequence_of(p.offsets, p.seqs, row, lane);
  const Sequence seq = sequence(p, b);
  if (row < seq.first || row >= seq.first + seq.n || (long long)seq.n * (p.heads / p.kv_heads) <= above) return;
  const long long keys = seq.keys - seq.n + (row - seq.first) + 1;
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

namespace {

// [pages][page_size][kv heads][head_dim], the middle dimensions in any order; box = 64 columns of one head x `box` keys of one page
bool pages_tmap(CUtensorMap* map, const bf16* base, const PagedAttention& p, int head_dim, long long page, long long row,
                long long head, int box) {
  EncodeFn fn = attn_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.kv_heads, 1ull << p.page_shift, (cuuint64_t)p.pages};
  // the stride of a dimension of one element is never used, but has to be a valid one
  auto bytes = [&](long long stride, cuuint64_t n) { return (cuuint64_t)(n == 1 ? head_dim : stride) * 2; };
  const cuuint64_t strides[3] = {bytes(head, dims[1]), bytes(row, dims[2]), bytes(page, dims[3])};
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1}, estr[4] = {1, 1, 1, 1};
  auto encode = [&] {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<bf16*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT && bind_primary_context()) r = encode();  // the first call of a thread
  return r == CUDA_SUCCESS;
}

// rows of the tile that takes the most rows a sequence can have here, 64 at most
int tile_rows(const PagedAttention& p) {
  const long long most = (long long)p.max_new * (p.heads / p.kv_heads);
  return most <= 16 ? 16 : most <= 32 ? 32 : 64;
}
int rows_ctas() { return 2 * attn_grid(1 << 20); }

template <typename C>
cudaError_t rows_launch(const PagedAttention& p, const Parts& parts, int ctas, cudaStream_t stream) {
  CUtensorMap tk, tv;
  const int box = std::min(kKeys, 1 << p.page_shift);
  if (!pages_tmap(&tk, p.k_pages, p, C::D, p.k_page, p.k_row, p.k_head, box) || !pages_tmap(&tv, p.v_pages, p, C::D, p.v_page, p.v_row, p.v_head, box))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> granted{0};
  const cudaError_t e = once_per_device(granted, [] {
    return cudaFuncSetAttribute(paged_rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_rows_kernel<C>, dim3(ctas), dim3(kRowsThreads), C::SMEM, stream, 0, tk, tv, p, parts, FastDiv(p.heads / p.kv_heads));
}

template <int D>
cudaError_t attention_launch(const PagedAttention& p, void* work, int* launches, cudaStream_t stream) {
  const int rows = tile_rows(p), ctas = rows_ctas();
  Parts parts;
  parts.rows = rows;
  parts.acc = reinterpret_cast<float*>(work);
  parts.ml = reinterpret_cast<float2*>(parts.acc + 2ll * ctas * rows * D);
  parts.share = reinterpret_cast<Share*>(parts.ml + 2ll * ctas * rows);
  cudaError_t e = rows == 16   ? rows_launch<Rows<D, 1>>(p, parts, ctas, stream)
                  : rows == 32 ? rows_launch<Rows<D, 2>>(p, parts, ctas, stream)
                               : rows_launch<Rows<D, 4>>(p, parts, ctas, stream);
  if (e != cudaSuccess) return e;
  *launches = 2;
  if ((long long)p.max_new * (p.heads / p.kv_heads) > rows) {
    const long long warps = (long long)p.tokens * p.heads;
    e = launch_pdl(paged_attention_kernel<D>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, 0, p, rows);
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  return launch_pdl(paged_join_kernel<D>, dim3(ctas, rows / 16), dim3(256), 0, stream, 0, p, parts, ctas);
}

}  // namespace

long long paged_attention_workspace(const PagedAttention& p, int head_dim) {
  const long long rows = tile_rows(p), ctas = rows_ctas();
  return 2 * ctas * rows * (head_dim * sizeof(float) + sizeof(float2)) + ctas * sizeof(Share);
}

cudaError_t paged_attention_launch(const PagedAttention& p, int head_dim, void* work, int* launches, cudaStream_t stream) {
  if (head_dim == 64) return attention_launch<64>(p, work, launches, stream);
  if (head_dim == 128) return attention_launch<128>(p, work, launches, stream);
  return cudaErrorInvalidValue;
}

}  // namespace dion
