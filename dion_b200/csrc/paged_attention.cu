// Causal attention of new tokens over a paged cache of keys and values:
//   out = softmax(scale q K[0..p]^T) V[0..p],   p = lengths[b] + i of row i of sequence b.
//
// The rows of a sequence that share a kv head (new tokens x heads of its group, token by token) make tiles of queries.  The keys
// are taken once per tile with the running maximum and sum of a softmax.  Few rows are bound by the bandwidth of the cache and go
// through mma.sync (paged_rows_kernel), many by the tensor core and the exponentials and go through tcgen05 (paged_chunk_kernel).
// Either way all keys of all tiles are dealt out evenly over the CTAs, whatever the lengths: a CTA's share may end inside a tile,
// whose parts a second kernel then joins.  Where the page table says that keys are few, a cluster of CTAs has a tile's instead and
// joins them itself.  Who has what follows from the sizes alone, so a call gives the same bits every time.
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

// What is worth a CTA.  One token over 1000 keys of 8 kv heads (us): 12.1 at 64, 12.9 at 128, 14.2 at 256; 6 heads of 777 keys 13.3,
// 13.6 and 14.7
constexpr int kShareCost = 64;

// How rows are put together: `group` query heads of one kv head (`subs` such groups make all of its heads, where these are more than
// a tile has rows) times `tokens` tokens are one tile of `height` rows, `tiles` of which go together.
struct Tiling {
  int height, tiles, group, subs, heads;          // heads: kv heads x subs
  int per, tokens, all;                           // tokens of a tile and of all `tiles`; query heads of a kv head
  int fixed;                                      // what such rows cost apart from their keys, in keys
  int side = 1;                                   // heads that CTAs next to one another have, see Walk
  FastDiv by_group;
  Tiling() = default;
  Tiling(const PagedAttention& p, int height_, int tiles_, int fixed_) : height(height_), tiles(tiles_), fixed(fixed_) {
    all = p.heads / p.kv_heads;
    subs = (all + height - 1) / height;
    group = (all + subs - 1) / subs;
    heads = p.kv_heads * subs;
    per = height / group;
    tokens = per * tiles;
    by_group = FastDiv(group);
  }
};

// A sequence of the call: rows first .. first + n, cached + n keys.  n = 0 where there is nothing to do or something is wrong.
struct Sequence {
  int first, n, cached;
  bool bad;
};
__device__ __forceinline__ Sequence sequence(const PagedAttention& p, int b) {
  const long long first = p.offsets[b], end = p.offsets[b + 1], cached = p.lengths[b], n = end - first;
  Sequence s{0, 0, 0, false};
  if (n == 0) return s;
  const long long most = min((long long)p.max_pages << p.page_shift, 0x7fffffffll - 1024);
  s.bad = first < 0 || n < 0 || end > p.tokens || cached < 0 || cached + n > most || n > p.max_new;
  if (!s.bad) s = Sequence{(int)first, (int)n, (int)cached, false};
  return s;
}

// An item is the rows of `tokens` tokens of one sequence and (part of a) kv head, with all keys that the last of them sees.  It costs
// as much as its keys and `fixed` more.  Costs have a closed form, so that any position in the line of all items is found without
// going through it.
struct Costs {
  int tokens, fixed, items;  // of a sequence, per head
  Sequence s;
  __device__ __forceinline__ Costs(const Sequence& s_, const Tiling& tl)
      : tokens(tl.tokens), fixed(tl.fixed), items((int)(((long long)s_.n + tl.tokens - 1) / tl.tokens)), s(s_) {}
  __device__ __forceinline__ int keys(int item) const { return (int)min((long long)s.cached + (item + 1ll) * tokens, (long long)s.cached + s.n); }
  __device__ __forceinline__ long long before(int item) const { return item * ((long long)s.cached + fixed) + (long long)tokens * item * (item + 1ll) / 2; }
  __device__ __forceinline__ long long head() const { return items > 0 ? before(items - 1) + fixed + s.cached + s.n : 0; }
};

// `side` CTAs next to one another have the same share of as many heads next to one another: in a page the rows of these lie side by
// side, and memory reads them at the same time.  100 sequences of 900 keys, 12 heads of 64, 59 us, a head after the other 71; 48
// prompts of up to 1024 tokens 98 and 108.
//
// Goes through a CTA's share: item `item` of head `head` (of tiling.heads) of sequence b, units begin .. end of its `units` units
// of K keys.  A share ends inside an item at a whole unit, or, where the item is small against the shares, at its nearer end.
// Every warp has one in shared memory, which its first lane moves on: in registers it would cost the softmax loops theirs.
template <int K>
struct Walk {
  long long to, at;  // positions in the line of all items: the share's end, this item's start
  int share;         // a share's cost, as far as it is comparable to an item's
  int b, head, item, begin, end, units, keys;
  int first, n, cached;  // of the sequence
  __device__ __forceinline__ bool valid() const { return at < to; }
  // the unit at position y of this item's cost
  __device__ __forceinline__ int cut(long long y, long long cost) const {
    if (4 * cost <= share) return 2 * y < cost ? 0 : units;
    return (int)(y * units / cost);
  }
  __device__ __forceinline__ void enter(const Tiling& tl, long long from) {
    keys = Costs(Sequence{first, n, cached, false}, tl).keys(item);
    units = (keys + K - 1) / K;
    const long long cost = (long long)keys + tl.fixed;
    begin = from <= at ? 0 : cut(from - at, cost);
    end = to >= at + cost ? units : cut(to - at, cost);
  }
  __device__ __forceinline__ void take(const Sequence& s) { first = s.first, n = s.n, cached = s.cached; }
  __device__ void next(const PagedAttention& p, const Tiling& tl) {
    do {
      at += (long long)keys + tl.fixed;
      if (at >= to) return;
      if ((++item) * (long long)tl.tokens >= n) {
        item = 0;
        if ((head += tl.side) >= tl.heads) {
          head -= tl.heads;
          Sequence s;
          do {
            if (++b >= p.seqs) {
              at = to;
              return;
            }
            s = sequence(p, b);
          } while (s.n == 0);
          take(s);
        }
      }
      enter(tl, at);
    } while (begin >= end);
  }
  // by a whole warp
  __device__ __forceinline__ void next(const PagedAttention& p, const Tiling& tl, int lane) {
    __syncwarp();
    if (lane == 0) next(p, tl);
    __syncwarp();
  }
};

template <int WARPS>
struct ShareScratch {  // of the block, in shared memory
  long long sums[WARPS], start;
  int b;
};

// Finds this CTA's share with the whole block and gives it to every warp.
template <int K, int WARPS>
__device__ __forceinline__ void my_share(const PagedAttention& p, const Tiling& tl, ShareScratch<WARPS>& scratch, Walk<K>& mine_) {
  constexpr int THREADS = 32 * WARPS;
  const int per = (p.seqs + THREADS - 1) / THREADS, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int lo = (int)min((long long)t * per, (long long)p.seqs), hi = min(lo + per, p.seqs);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += Costs(sequence(p, b), tl).head() * (tl.heads / tl.side);
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scratch.sums[warp] = upto;
  if (t == 0) scratch.b = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) upto += scratch.sums[i];
    total += scratch.sums[i];
  }
  const int shares_most = gridDim.x / tl.side, nth = blockIdx.x / tl.side;
  const long long shares = max(1ll, min((long long)shares_most, total / kShareCost));
  const long long each = total / shares, rest = total - each * shares;
  long long from = 0, to = 0;
  if (nth < shares) {  // total * nth / shares without a product of 64 x 64 bits
    from = each * nth + rest * nth / shares;
    to = each * (nth + 1) + rest * (nth + 1) / shares;
  }
  if (from < to && upto - mine <= from && from < upto) {  // the thread whose sequences hold the start
    long long at = upto - mine;
    for (int b = lo; b < hi; ++b) {
      const long long cost = Costs(sequence(p, b), tl).head() * (tl.heads / tl.side);
      if (from < at + cost) {
        scratch.b = b;
        scratch.start = at;
        break;
      }
      at += cost;
    }
  }
  __syncthreads();
  if (lane == 0) {
    Walk<K> w{};
    w.b = scratch.b;
    if (w.b >= 0) {
      w.to = to;
      w.at = scratch.start;
      w.share = (int)min(each, 0x7fffffffll);
      const Sequence s = sequence(p, w.b);
      w.take(s);
      const Costs c(s, tl);
      const int before = (int)((from - w.at) / c.head());
      w.head = before * tl.side + blockIdx.x % tl.side;
      w.at += before * c.head();
      int low = 0, high = c.items;  // the item that holds the start
      while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (c.before(mid) <= from - w.at) low = mid;
        else high = mid;
      }
      w.item = low;
      w.at += c.before(low);
      w.enter(tl, from);
      if (w.begin >= w.end) w.next(p, tl);
    }
    mine_ = w;
  }
  __syncwarp();
}

// What a CTA leaves for the join.  Slot 2c holds its first item where an earlier CTA has begun it, slot 2c + 1 its last one where a
// later CTA ends it.
struct Share {
  int b, head, item;  // in slot 2c + 1; b = -1: none
  short continues;    // slot 2c is filled; -1: the share has not one unit, and the slot says that it has no part in anything
  short ends;         // slot 2c's item ends here
};
struct Parts {
  float* acc;    // [slot][rows of an item][head_dim], not normalised
  float2* ml;    // [slot][rows of an item]: maximum (log2 units) and sum
  Share* share;  // per CTA
  int cluster, items;  // where a cluster has an item: its CTAs, and items of a sequence and head
};

// Row r of an item: its token in the sequence and its query head; false where there is none
__device__ __forceinline__ bool row_of(const PagedAttention& p, const Tiling& tl, int n, int head, int item, int tile, int r, int& token,
                                       int& h) {
  const int per = tl.tokens / tl.tiles, i = tl.by_group(r), kv = tl.subs == 1 ? head : head / tl.subs, sub = head - kv * tl.subs;
  const int all = p.heads / p.kv_heads, in_group = sub * tl.group + (r - i * tl.group);
  token = item * tl.tokens + tile * per + i;
  h = kv * all + in_group;
  return i < per && token < n && in_group < all;
}

// ---------------------------------------------------------------------------------- few rows per kv head: mma.sync

constexpr int kKeys = 64;               // keys of a stage
// What an item costs apart from its keys, in keys: the first load's way, the warps' join, the result.  200 sequences of up to 200
// keys, 32 heads on 8 (us): 79 at 0, 34 at 128, 28 at 256, 30 at 512; where all are long it makes no difference.
constexpr int kRowsFixed = 256;
constexpr int kFewCluster = 8;        // CTAs of a cluster that has one item, at most
constexpr int kFewItems = 1 << 20;   // items of such a launch, at most
constexpr int kRowsThreads = 32 * 5;    // four warps of products and one that loads

template <int D_, int WM_, bool FEW_>
struct Rows {
  static constexpr int D = D_, WM = WM_, WK = 4 / WM, TR = 16 * WM;  // warps along the rows and along the keys, rows of a tile
  static constexpr bool FEW = FEW_;  // an item per cluster
  static constexpr int PANELS = D / 64, PANEL = kKeys * 128, STAGE = 2 * PANELS * PANEL;  // bytes; K panels, then V panels
  static constexpr int STAGES = D == 128 ? 3 : FEW ? 4 : 6;
  static constexpr int EXCHANGE = WK > 1 ? 2 * 16 * D * 4 : 0;  // accumulators of two warps on their way to their neighbours
  static constexpr int SMEM = STAGES * STAGE + EXCHANGE + 1024;
  static_assert(SMEM <= 115712, "two CTAs per SM");
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

__device__ __forceinline__ float4 remote4(const float* v, int rank) {
  float4 r;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
               : "r"(mapa_shared(smem_u32(v), (uint32_t)rank))
               : "memory");
  return r;
}
__device__ __forceinline__ float2 remote2(const void* v, int rank) {
  float2 r;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(mapa_shared(smem_u32(v), (uint32_t)rank)) : "memory");
  return r;
}

// Writes zeros to rows that are nobody's (behind the last sequence, of wrong ones) and reports what is wrong with the sequences: the
// part of block `block` of `blocks`, by threads `t` of `threads`.
template <int D>
__device__ __forceinline__ void nobodys_rows(const PagedAttention& p, int block, int blocks, int t, int threads) {
  auto clear = [&](long long lo, long long hi) {
    lo = max(lo, 0ll);
    hi = min(hi, (long long)p.tokens);
    const long long per_row = (long long)p.heads * D / 8;
    for (long long i = lo * per_row + t; i < hi * per_row; i += threads) reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
  };
  for (int b = block; b < p.seqs; b += blocks) {
    if (sequence(p, b).bad) {
      if (t == 0) bad_argument(p.status);
      clear(p.offsets[b], p.offsets[b + 1]);
    }
  }
  if (block == 0 && t == 0 && p.offsets[0] != 0) bad_argument(p.status);
  for (long long r = max(0ll, (long long)p.offsets[p.seqs]) + block; r < p.tokens; r += blocks) clear(r, r + 1);
}

// Bound by the bandwidth of the cache: 64 keys are 32 KB (head dimension 128), which an SM gets in 1400 cycles, and take four
// warps some 600.  So the legacy products, whose tiles are 16 rows high, do: the rows of single tokens fill no more.  A warp loads
// 64 keys a stage by TMA, the boxes of several pages where they are smaller; where the rows fit one 16-row tile the four others
// take 16 keys each and join their sums per item, else they share the keys and have rows of their own.  Two caches of 120000 keys, 8
// kv heads of 128: 152 us, 6.4 TB/s; 64 of up to 8000 139 us, 6.1 TB/s.
//
// FEW: a cluster has one item, its CTAs equal parts of the keys, and the parts are joined over the cluster's shared memory.  That
// saves the second kernel where items are short; what counts there is the chain of latencies.
template <typename C>
__global__ void __launch_bounds__(kRowsThreads, 2)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const PagedAttention p,
                  const Parts parts, const __grid_constant__ Tiling tl) {
  constexpr int D = C::D, WK = C::WK, TR = C::TR;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* exchange = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE + C::EXCHANGE);
  uint64_t* empty = full + C::STAGES;
  auto* scratch = reinterpret_cast<ShareScratch<kRowsThreads / 32>*>(empty + C::STAGES);
  auto* walks = reinterpret_cast<Walk<kKeys>*>(scratch + 1);
  float2* stats = reinterpret_cast<float2*>(walks + kRowsThreads / 32);  // [warp][16 rows]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(stats + 4 * 16);
  static_assert(C::STAGES * 16 + sizeof(*scratch) + sizeof(*walks) * kRowsThreads / 32 + 4 * 16 * sizeof(float2) + 4 <= 1024);
  const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {  // the 128-byte swizzle repeats every 1024 bytes
    if (threadIdx.x == 0) {
      bad_argument(p.status);
      if (!C::FEW) parts.share[blockIdx.x] = Share{-1, 0, 0, -1, 0};
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
  Walk<kKeys>& w = walks[warp];
  const int rank = C::FEW ? (int)blockIdx.x % parts.cluster : 0;
  if constexpr (C::FEW) {
    if (lane == 0) {
      Walk<kKeys> mine{};
      const int nth = (int)blockIdx.x / parts.cluster, seq_item = nth / tl.heads;
      mine.head = nth - seq_item * tl.heads;
      mine.b = seq_item / parts.items;
      mine.item = seq_item - mine.b * parts.items;
      const Sequence s = sequence(p, mine.b);
      mine.take(s);
      const Costs c(s, tl);
      if (mine.item < c.items) {
        mine.to = 1;  // valid
        mine.keys = c.keys(mine.item);
        mine.units = (mine.keys + kKeys - 1) / kKeys;
        mine.begin = (int)((long long)mine.units * rank / parts.cluster);
        mine.end = (int)((long long)mine.units * (rank + 1) / parts.cluster);
      }
      w = mine;
    }
    __syncthreads();
  } else {
    my_share(p, tl, *scratch, w);
  }
  Ring<C::STAGES> ring;

  if (warp == 4) {
    // ------------------------------------------------------------------ loads
    const int shift = p.page_shift, box = min(kKeys, 1 << shift), boxes = kKeys / box;
    for (; w.valid(); w.next(p, tl, lane)) {
      const int* table = p.page_table + (long long)w.b * p.table_pitch;
      const int used = (int)(((long long)w.keys + (1 << shift) - 1) >> shift);
      int held = 0, have = 0, page = 0;  // lane i: page held + i, for i < have
      for (int u = w.begin; u < w.end; ++u) {
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
      if (C::FEW || __any_sync(0xffffffffu, *abort_flag != 0)) break;
    }
    if (C::FEW) nobodys_rows<D>(p, blockIdx.x, gridDim.x, lane, 32);
  } else {
    // ------------------------------------------------------------------ products
    // A wait that gives up raises the abort flag and the warp goes on without waiting, so that the barriers of the four are met.
    const int wm = warp % C::WM, wk = warp / C::WM;
    constexpr int KG = kKeys / WK / 16;  // groups of 16 keys that this warp has in a stage
    const int key0 = wk * (kKeys / WK), quad = lane >> 2, pair = (lane & 3) * 2;
    const float scale = p.scale * 1.4426950408889634f;
    bool dead = false;
    Share share{-1, 0, 0, -1, 0};
    bool first_item = true;
    for (; w.valid(); w.next(p, tl, lane)) {
      const int least = w.cached + w.item * tl.tokens + 1;  // keys that the first token sees
      // queries of rows quad and quad + 8, and how many keys these see
      uint32_t q[D / 16][4];
      int sees[2];
      long long to[2];  // their rows of the result
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int token, h;
        const bool there = row_of(p, tl, w.n, w.head, w.item, 0, wm * 16 + quad + 8 * i, token, h);
        sees[i] = there ? w.cached + token + 1 : least;
        to[i] = there ? ((long long)(w.first + token) * p.heads + h) * D : -1;
        if (!there) token = w.item * tl.tokens, h = w.head / tl.subs * (p.heads / p.kv_heads);  // a row that exists
        const bf16* src = p.q + (w.first + token) * p.q_token + h * p.q_head + pair;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          q[kk][i] = *reinterpret_cast<const uint32_t*>(src + kk * 16);
          q[kk][2 + i] = *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8);
        }
      }
      float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      for (int u = w.begin; u < w.end; ++u) {
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
        if (at + KG * 16 > least) {  // beyond what the first token sees
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
        const bool ragged = at + KG * 16 > w.keys;  // what lies behind the last key may be no numbers: taken as zeros
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const uint32_t a[4] = {pr[2 * g][0], pr[2 * g][1], pr[2 * g + 1][0], pr[2 * g + 1][1]};
          const int left = w.keys - (at + g * 16) - pair;  // of the keys from this lane's first on
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
      const bool starts = w.begin == 0, ends = w.end == w.units;
      if (C::FEW && parts.cluster > 1) {
        products_sync();  // nobody reads the ring or the statistics any more: the sums go there
        if (wk == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = wm * 16 + quad + 8 * i;
            if ((lane & 3) == 0) stats[r] = make_float2(m[i], l[i]);
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<float2*>(reinterpret_cast<float*>(smem) + r * D + c * 8 + pair) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
          }
        }
        break;
      }
      if (wk == 0) {
        if (starts && ends) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (to[i] < 0) continue;
            const float inv = 1.f / l[i];  // the row sees a key; no numbers, or none but -infinity, stay no numbers
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
      if (starts && !ends) share.b = w.b, share.head = w.head, share.item = w.item;
      if (first_item) share.continues = !starts, share.ends = ends;
      first_item = false;
      if (C::FEW) break;
    }
    if (!C::FEW) {
      if (threadIdx.x == 0) parts.share[blockIdx.x] = share;
      if (share.continues < 0 && threadIdx.x < TR) parts.ml[2ll * blockIdx.x * TR + threadIdx.x] = make_float2(-INFINITY, 0.f);
    }
  }
  if (C::FEW && parts.cluster > 1 && w.valid()) {  // the same in all CTAs of the cluster
    cluster_sync_all();
    for (int r = rank + parts.cluster * warp; r < tl.height; r += parts.cluster * (kRowsThreads / 32)) {
      int token, h;
      if (!row_of(p, tl, w.n, w.head, w.item, 0, r, token, h)) continue;
      const float2 t = lane < parts.cluster ? remote2(&stats[r], lane) : make_float2(-INFINITY, 0.f);
      float top = t.x;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = __shfl_sync(0xffffffffu, top, 0);  // of the first eight lanes; the row sees a key, so some part has one
      const float f = fast_exp2(t.x - top);
      float sum = t.y * f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = 1.f / __shfl_sync(0xffffffffu, sum, 0);
      const float* acc = reinterpret_cast<const float*>(smem) + r * D + lane * (D / 32);
      float v[D / 32] = {};
#pragma unroll 8
      for (int k = 0; k < parts.cluster; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        if constexpr (D == 128) {
          const float4 a = remote4(acc, k);
          v[0] += a.x * fk, v[1] += a.y * fk, v[2] += a.z * fk, v[3] += a.w * fk;
        } else {
          const float2 a = remote2(acc, k);
          v[0] += a.x * fk, v[1] += a.y * fk;
        }
      }
      bf16* dst = p.out + ((long long)(w.first + token) * p.heads + h) * D + lane * (D / 32);
#pragma unroll
      for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(v[i] * inv, v[i + 1] * inv);
    }
    cluster_sync_all();  // nobody reads another's shared memory after this
  }
  __syncthreads();
  if (*abort_flag != 0) {
    // a wait gave up: let copies that are still in flight land before the CTA retires
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
}

// CTAs c, c + side ... have the parts of the item that CTA c has begun: how many come after c, up to the one that ends it.  By a whole
// warp; any answer, in bounds, where c has begun none.
__device__ __forceinline__ int parts_after(const Parts& parts, const Share& mine, int c, int side, int ctas, int lane) {
  int last = 0;
  for (bool more = true; more;) {
    const int i = c + (last + 1 + lane) * side;
    const Share s = parts.share[min(i, ctas - 1)];
    const unsigned at = __ballot_sync(0xffffffffu, i >= ctas || s.continues == 0 || (s.continues > 0 && s.ends));
    more = at == 0 && mine.b >= 0;
    last += more ? 32 : __ffs(at);
  }
  return min(last, (ctas - 1 - c) / side);
}
template <int E>
__device__ __forceinline__ void load_columns(const float* from, float (&v)[E]) {
  if constexpr (E == 4) {
    const float4 x = *reinterpret_cast<const float4*>(from);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const float2 x = *reinterpret_cast<const float2*>(from);
    v[0] = x.x, v[1] = x.y;
  }
}

// Joins the parts of items that several CTAs had and sees to nobody's rows; for few rows, which come in many parts (a cache of 4000
// keys over the whole GPU in 30).  Block (c, y) has the item that CTA c began, and of its rows every gridDim.y-th, whose parts the
// WARPS warps share.  Bound by latency: what the next step needs is loaded before this one has decided whether, and the code is
// kept short, as every call fetches it anew.
template <int D, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) paged_join_kernel(const PagedAttention p, const Parts parts, const __grid_constant__ Tiling tl) {
  constexpr int E = D / 32;  // columns of a lane
  __shared__ float sums[WARPS][D + 2];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x, ctas = gridDim.x, rows = tl.height, side = tl.side;
  const Share mine = parts.share[c];
  const int last = parts_after(parts, mine, c, side, ctas, lane);
  if (mine.b >= 0) {
    const Sequence s = sequence(p, mine.b);
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
      int token, h;
      if (!row_of(p, tl, s.n, mine.head, mine.item, 0, r, token, h)) continue;  // the whole block
      float top = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      auto slot = [&](int nth) { return (2 * (c + (long long)nth * side) + (nth == 0 ? 1 : 0)) * rows + r; };
      // this warp's parts are numbers warp, warp + WARPS ..., 32 at a time
      for (int base = warp; base <= last; base += 32 * WARPS) {
        const int nth = base + lane * WARPS, n = min(32, (last - base) / WARPS + 1);
        const float2 t = nth <= last ? parts.ml[slot(nth)] : make_float2(-INFINITY, 0.f);
        float most = t.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float top2 = fmaxf(top, most), neg = top2 == -INFINITY ? 0.f : -top2, f = fast_exp2(top + neg), w = fast_exp2(t.x + neg);
        sum = sum * f + t.y * w;  // of this lane's parts
        top = top2;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll 1
        for (int k = 0; k < n; k += 4) {
          float v[4][E];
#pragma unroll
          for (int j = 0; j < 4; ++j) load_columns<E>(parts.acc + slot(base + min(k + j, n - 1) * WARPS) * D + lane * E, v[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float wj = __shfl_sync(0xffffffffu, w, (k + j) & 31);
            if (k + j < n && wj > 0.f) {  // a part that saw none of the row's keys has nothing written
#pragma unroll
              for (int e = 0; e < E; ++e) acc[e] += wj * v[j][e];
            }
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sums[warp][D] = top, sums[warp][D + 1] = sum;
#pragma unroll
      for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = acc[e];
      __syncthreads();
      if (warp == 0) {
        const float mine_top = top;
#pragma unroll 1
        for (int i = 1; i < WARPS; ++i) top = fmaxf(top, sums[i][D]);
        float f = fast_exp2(mine_top - top);
        sum *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll 1
        for (int i = 1; i < WARPS; ++i) {
          f = fast_exp2(sums[i][D] - top);
          sum += sums[i][D + 1] * f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += sums[i][lane * E + e] * f;
        }
        const float inv = 1.f / sum;  // no number where a part's sum is none, whatever its weight
        bf16* dst = p.out + ((long long)(s.first + token) * p.heads + h) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
      }
      __syncthreads();
    }
  }
  if (blockIdx.y == 0) nobodys_rows<D>(p, c, ctas, threadIdx.x, 32 * WARPS);
}

// The same for many rows, which come in two or three parts: a warp takes four rows at a time, their maxima and sums of up to eight
// parts in one load, so that they are all under way at once.  With the kernel above it, 2048 tokens over 6000 cached, two sequences, 32
// heads on 8 of 128, take 415 us, 421 with a row after the other; with blocks of eight warps instead of four a call that has nothing
// to join took 227 us instead of 208.
constexpr int kJoinWarps = 4, kJoinRows = 4;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_many_kernel(const PagedAttention p, const Parts parts, const __grid_constant__ Tiling tl) {
  constexpr int E = D / 32, R = kJoinRows, K = 32 / R;  // columns of a lane, rows of a warp, parts at a time
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x, ctas = gridDim.x, rows = tl.height * tl.tiles, side = tl.side;
  const Share mine = parts.share[c];
  const int last = parts_after(parts, mine, c, side, ctas, lane);
  if (mine.b >= 0) {
    const Sequence s = sequence(p, mine.b);
    for (int r0 = (blockIdx.y * kJoinWarps + warp) * R; r0 < rows; r0 += gridDim.y * kJoinWarps * R) {
      auto slot = [&](int nth) { return (2 * (c + (long long)nth * side) + (nth == 0 ? 1 : 0)) * rows + r0; };
      float top = -INFINITY, sum = 0.f, acc[R][E];  // top and sum of row r0 + lane / K, this lane's parts
#pragma unroll
      for (int j = 0; j < R; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[j][e] = 0.f;
      for (int base = 0; base <= last; base += K) {
        const int nth = base + lane % K, n = min(K, last - base + 1);
        const float2 t = nth <= last ? parts.ml[slot(nth) + lane / K] : make_float2(-INFINITY, 0.f);
        float most = t.x;
#pragma unroll
        for (int o = K / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float top2 = fmaxf(top, most), neg = top2 == -INFINITY ? 0.f : -top2, f = fast_exp2(top + neg), w = fast_exp2(t.x + neg);
        sum = sum * f + t.y * w;
        top = top2;
        if (base > 0) {
#pragma unroll
          for (int j = 0; j < R; ++j) {
            const float fj = __shfl_sync(0xffffffffu, f, j * K);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[j][e] *= fj;
          }
        }
#pragma unroll 2
        for (int k = 0; k < n; ++k) {
          float v[R][E];
#pragma unroll
          for (int j = 0; j < R; ++j) load_columns<E>(parts.acc + (slot(base + k) + j) * D + lane * E, v[j]);
#pragma unroll
          for (int j = 0; j < R; ++j) {
            const float wj = __shfl_sync(0xffffffffu, w, j * K + k);
            if (wj > 0.f) {  // a part that saw none of the row's keys has nothing written
#pragma unroll
              for (int e = 0; e < E; ++e) acc[j][e] += wj * v[j][e];
            }
          }
        }
      }
#pragma unroll
      for (int o = K / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = 1.f / sum;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int r = r0 + j;
        const float f = __shfl_sync(0xffffffffu, inv, j * K);
        int token, h;
        if (!row_of(p, tl, s.n, mine.head, mine.item, r / kBM, r % kBM, token, h)) continue;
        bf16* dst = p.out + ((long long)(s.first + token) * p.heads + h) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(acc[j][e] * f, acc[j][e + 1] * f);
      }
    }
  }
  if (blockIdx.y == 0) nobodys_rows<D>(p, c, ctas, threadIdx.x, 32 * kJoinWarps);
}

// ---------------------------------------------------------------------------------- many rows: tcgen05

// As kRowsFixed.  48 prompts of up to 1024 tokens, 12 heads of 64 (us): 147 at 0, 116 at 128, 112 at 256, 108.5 at 384, 110 at 512
constexpr int kChunkFixed = 384;
constexpr int kChunkThreads = 32 * 12;  // loads; products of either query tile; a spare; four softmax warps per query tile

template <int D>
struct Chunk {
  static constexpr int PANELS = D / 64;           // 128-byte panels along the head dimension
  static constexpr int TILE_BYTES = kBM * D * 2;  // 128 rows of Q, K or V
  static constexpr int K_STAGES = D == 128 ? 3 : 4, V_STAGES = D == 128 ? 2 : 4;
  static constexpr int SMEM = (2 + K_STAGES + V_STAGES) * TILE_BYTES + 1536;
  // tensor memory: S and O of both query tiles; D = 64 has room for P beside S, D = 128 writes P over S
  static constexpr bool P_APART = D == 64;
  static constexpr int S_COL = 0, O_COL = 2 * kBM, P_COL = P_APART ? 2 * kBM + 2 * D : S_COL;
  static constexpr int P_TILE = P_APART ? 64 : kBM;  // columns from one query tile's P to the other's
  static constexpr int TMEM_COLS = 512;
  static_assert(P_COL + 2 * 64 <= TMEM_COLS && O_COL + 2 * D <= TMEM_COLS && SMEM <= 232448, "one CTA per SM");
};

// Units of an item that its query tile x has to do: those of this share up to the last one that a row of the tile sees
__device__ __forceinline__ int tile_end(const Walk<kBM>& w, const Tiling& tl, int x) {
  const int per = tl.tokens / 2, first = w.item * tl.tokens + x * per;
  if (first >= w.n) return w.begin;
  const int sees = w.cached + min(first + per, w.n);
  return max(w.begin, min(w.end, (sees + kBM - 1) / kBM));
}

// One CTA per SM goes through items of two query tiles of 128 rows, which share the K and V tiles; each has four softmax warps with
// a query row per thread and a warp that issues its products, so that one tile's exponentials run under the other's products.  K
// and V come page by page; keys behind the last one are masked and their values, which may be no numbers, replaced by zeros in
// shared memory by the softmax warps before they hand on the weights.
//
// A unit of 128 keys of both tiles takes 3200 cycles for heads of 64 and 4100 of 128 (2048 tokens over 6000 cached, two sequences, 32
// heads on 8 of 128: 415 us, 1.13 PFLOP/s).  Its exponentials take 2048 of the special function unit, its products 1024 and 2048
// of the tensor core; what is on top is the chain of a tile: at 128 its next S waits for P V, as P lies over S, 1700 cycles of
// which 1024 are products, and at 64 both tiles' exponentials run at the same time.  Measured and not kept (cycles a unit, 64 / 128):
// a quarter of the exponentials by a polynomial (3200 / 4700, the multiply-adds take 14 cycles a value of a warp, the special function
// unit 8), two threads for a row (3400 / 5500), P V in two halves (3200 / 4800 with both tiles), the next scores
// loaded during the exponentials (3400), two CTAs with a tile each (3400), a lock between the tiles' exponentials (3800 / 3600).
template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const PagedAttention p, const Parts parts, const __grid_constant__ Tiling tl) {
  using C = Chunk<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;  // two tiles
  uint8_t* sK = sQ + 2 * C::TILE_BYTES;
  uint8_t* sV = sK + C::K_STAGES * C::TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + C::V_STAGES * C::TILE_BYTES);
  uint64_t* q_full = bars;        // one per query tile, as the next five
  uint64_t* q_empty = bars + 2;
  uint64_t* s_full = bars + 4;
  uint64_t* s_free = bars + 6;    // four warps: S is in registers (P_APART)
  uint64_t* p_full = bars + 8;    // four warps
  uint64_t* pv_done = bars + 10;  // O += P V retired: O stable, P free
  uint64_t* k_full = bars + 12;   // K_STAGES each
  uint64_t* k_empty = k_full + C::K_STAGES;
  uint64_t* v_full = k_empty + C::K_STAGES;  // V_STAGES each
  uint64_t* v_empty = v_full + C::V_STAGES;
  uint64_t* bars_end = v_empty + C::V_STAGES;
  auto* scratch = reinterpret_cast<ShareScratch<kChunkThreads / 32>*>(bars_end);
  auto* walks = reinterpret_cast<Walk<kBM>*>(scratch + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(walks + kChunkThreads / 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((12 + 2 * (C::K_STAGES + C::V_STAGES)) * 8 + sizeof(*scratch) + sizeof(*walks) * kChunkThreads / 32 + 8 <= 1536);

  const int warp = (int)warp_uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {  // the 128-byte swizzle repeats every 1024 bytes
    if (threadIdx.x == 0) {
      bad_argument(p.status);
      parts.share[blockIdx.x] = Share{-1, 0, 0, -1, 0};
    }
    return;
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    for (uint64_t* b = bars; b < bars_end; ++b)
      mbar_init(b, (b >= s_free && b < pv_done) ? 4 : ((b >= k_empty && b < v_full) || b >= v_empty) ? 2 : 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  pdl_trigger();
  pdl_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  Walk<kBM>& w = walks[warp];
  tc_fence_before();
  my_share(p, tl, *scratch, w);  // synchronises the block
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);
  const int per = tl.tokens / 2;  // tokens of a query tile

  if (warp < 4) {
    give_registers<96, 200>();
    if (warp == 0) {
      // ---------------------------------------------------------------- loads
      const int shift = p.page_shift, box = min(kBM, 1 << shift), boxes = kBM / box;
      Ring<C::K_STAGES> ks;
      Ring<C::V_STAGES> vs;
      int nq[2] = {0, 0};  // loads of each query tile's buffer
      bool ok = true;
      auto free_slot = [&](uint64_t* bar, uint32_t parity) {  // the same answer in all lanes
        const bool got = mbar_wait(bar, parity, abort_flag);
        ok = __all_sync(0xffffffffu, got);
        return ok;
      };
      for (; ok && w.valid(); w.next(p, tl, lane)) {
        const int* table = p.page_table + (long long)w.b * p.table_pitch;
        const int used = (int)(((long long)w.keys + (1 << shift) - 1) >> shift);
        const int kv = w.head / tl.subs, h0 = kv * (p.heads / p.kv_heads) + (w.head - kv * tl.subs) * tl.group;
        int held = 0, have = 0, page = 0;  // lane i: page held + i, for i < have
        for (int x = 0; x < 2 && ok; ++x) {
          if (tile_end(w, tl, x) == w.begin) continue;
          if (!free_slot(&q_empty[x], (nq[x] & 1) ^ 1u)) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[x], per * tl.group * D * 2);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_3d(sQ + x * C::TILE_BYTES + c * (kBM * 128), &tmap_q, &q_full[x], c * 64, h0, w.first + w.item * tl.tokens + x * per);
          }
          ++nq[x];
        }
        for (int u = w.begin; ok && u < w.end; ++u) {
          const int key = u * kBM, first = key >> shift, count = min(boxes, used - first), at = key & ((1 << shift) - 1);
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
          auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar) {
            if (lane == 0) mbar_arrive_expect_tx(bar, count * box * D * 2);
            __syncwarp();
            if (lane < count) {
#pragma unroll
              for (int c = 0; c < C::PANELS; ++c) tma_load_4d(dst + c * (kBM * 128) + lane * box * 128, map, bar, c * 64, kv, at, mine);
            }
          };
          if (!free_slot(&k_empty[ks.s], ks.ph ^ 1u)) break;
          load(sK + ks.s * C::TILE_BYTES, &tmap_k, &k_full[ks.s]);
          if (!free_slot(&v_empty[vs.s], vs.ph ^ 1u)) break;
          load(sV + vs.s * C::TILE_BYTES, &tmap_v, &v_full[vs.s]);
          ks.next();
          vs.next();
        }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        atomicCAS(p.status, 0, kStatusProducerTimeout);
      }
    } else if (warp < 3) {
      // ---------------------------------------------------------------- S = Q K^T and O += P V of one query tile
      if (elect_one()) {
        const int x = warp - 1;
        constexpr uint32_t idesc = make_instr_desc(1, kMajorK, kMajorMN, kBM, D);
        const DescHalves dq_ = desc_halves(smem_u32(sQ) + x * C::TILE_BYTES, 16, 1024), dk_ = desc_halves(smem_u32(sK), 16, 1024);
        const DescHalves dv_ = desc_halves(smem_u32(sV), kBM * 128, 1024);
        const uint32_t s_col = tmem_base + C::S_COL + x * kBM, p_col = tmem_base + C::P_COL + x * C::P_TILE;
        const uint32_t o_col = tmem_base + C::O_COL + x * D;
        bool ok = true;
        Ring<C::K_STAGES> ks;
        Ring<C::V_STAGES> vs;
        uint32_t ph = 0;  // of the unit whose P is awaited
        uint32_t nq = 0;  // query tiles so far
        auto issue_s = [&](int u, int end) {  // S of unit u of the item at hand
          ok = ok && mbar_wait(&k_full[ks.s], ks.ph, abort_flag) && (u > w.begin || mbar_wait(&q_full[x], nq & 1, abort_flag));
          if (!ok) return;
          tc_fence_after();
          scores<D, false>(s_col, dq_, 0, dk_, ks.s * C::TILE_BYTES);
          umma_commit(&s_full[x]);
          umma_commit(&k_empty[ks.s]);
          if (u == end - 1) {
            umma_commit(&q_empty[x]);
            ++nq;
          }
          ks.next();
        };
        auto skip = [&]() {  // a pair of K and V tiles that this query tile does not see: passed on once it has arrived
          ok = ok && mbar_wait(&k_full[ks.s], ks.ph, abort_flag);
          if (ok) mbar_arrive(&k_empty[ks.s]);
          ok = ok && mbar_wait(&v_full[vs.s], vs.ph, abort_flag);
          if (ok) mbar_arrive(&v_empty[vs.s]);
          ks.next();
          vs.next();
        };
        for (; ok && w.valid(); w.next(p, tl)) {
          const int end = tile_end(w, tl, x);
          if (end > w.begin) issue_s(w.begin, end);  // the S before has been read: P of it has been multiplied
          for (int u = w.begin; u < end && ok; ++u) {
            if (C::P_APART && u + 1 < end) {
              ok = mbar_wait(&s_free[x], ph, abort_flag);
              issue_s(u + 1, end);
            }
            ok = ok && mbar_wait(&v_full[vs.s], vs.ph, abort_flag) && mbar_wait(&p_full[x], ph, abort_flag);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kBM / 16; ++kk)
              umma_ts_h(o_col, p_col + kk * 8, dv_, vs.s * C::TILE_BYTES + kk * (16 * 128), idesc, (u > w.begin || kk > 0) ? 1u : 0u);
            umma_commit(&pv_done[x]);
            umma_commit(&v_empty[vs.s]);
            vs.next();
            if (!C::P_APART && u + 1 < end) issue_s(u + 1, end);  // over the P just read: the tensor core keeps the order
            ph ^= 1u;
          }
          for (int u = end; u < w.end && ok; ++u) skip();
        }
        if (!ok) {
          *abort_flag = 1;
          atomicCAS(p.status, 0, kStatusMmaTimeout);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, stores
    // Quadrant = warp & 3 (query rows), x = which query tile.  A wait that gives up raises the abort flag for all roles
    // and the warp goes on (its lanes stay together); nothing is stored then.
    take_registers<96, 200>();
    const int quad = warp & 3;
    const int x = (warp - 4) >> 2;
    const int row_in_tile = quad * 32 + lane;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_col = lane_base + C::S_COL + x * kBM, p_col = lane_base + C::P_COL + x * C::P_TILE;
    const uint32_t o_col = C::O_COL + x * D;
    const float scale_log2 = p.scale * 1.4426950408889634f;
    const f32x2 s2 = pack2(scale_log2, scale_log2);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!mbar_wait(bar, parity, abort_flag)) *abort_flag = 1;
      __syncwarp();  // the tensor-memory accesses that follow take the whole warp at once
    };
    uint32_t ph = 0;      // of the unit at hand: s_full, s_free, p_full, pv_done
    uint32_t passed = 0;  // units of the items before
    Share share{-1, 0, 0, -1, 0};
    bool first_item = true;
    for (; w.valid(); w.next(p, tl, lane)) {
      const int end = tile_end(w, tl, x), keys = w.keys;
      const int first = w.item * tl.tokens + x * per;
      const int least = w.cached + first + 1;                                // keys that the first row sees
      const int sees = w.cached + min(first + tl.by_group(row_in_tile), w.n - 1) + 1;  // and this one
      float m_used = -INFINITY;  // reference max of the exponentials accumulated so far (log2 domain)
      float l = 0.f;
      for (int u = w.begin; u < end; ++u) {
        wait(&s_full[x], ph);
        tc_fence_after();
        float sc[kBM];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_col + c * 32, *reinterpret_cast<float(*)[32]>(&sc[c * 32]));
        tmem_ld_wait();
        if (C::P_APART) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[x]);
        }
        if ((u + 1) * kBM > least) {
          const int mine = sees - u * kBM;
#pragma unroll
          for (int i = 0; i < kBM; ++i)
            if (i >= mine) sc[i] = -INFINITY;
        }
        if ((u + 1) * kBM > keys) {  // what lies behind the last key may be no numbers
          const uint32_t nth = passed + (uint32_t)(u - w.begin), stage = nth % C::V_STAGES;
          wait(&v_full[stage], (nth / C::V_STAGES) & 1);
          if (row_in_tile >= keys - u * kBM) {
#pragma unroll
            for (int c = 0; c < C::PANELS * 8; ++c)
              *reinterpret_cast<uint4*>(sV + stage * C::TILE_BYTES + (c >> 3) * (kBM * 128) + row_in_tile * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_shared();
        }
        // row maximum of the raw scores (the scale is positive), four independent chains
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kBM; i += 8) {
#pragma unroll
          for (int t = 0; t < 4; ++t) mx4[t] = fmaxf(mx4[t], fmaxf(sc[i + 2 * t], sc[i + 2 * t + 1]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
        const float m_new = fmaxf(m_used, mx);
        const bool need = u == w.begin || m_new - m_used > kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          if (u > w.begin) {
            // O may only be touched between two products: the one before must have retired, the next one cannot start
            // before this warp delivered its P
            wait(&pv_done[x], ph ^ 1u);
            tc_fence_after();
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld_32x32(lane_base + o_col + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= alpha;
              tmem_st_32x32(lane_base + o_col + c * 32, o);
            }
            tmem_st_wait();
          }
          m_used = m_new;
        }
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
        const f32x2 nm2 = pack2(neg_m, neg_m);
        f32x2 sums[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        // exponentials, packed to bf16 pairs; their sum is that of the unrounded ones
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float e0, e1;
            unpack2(fma2(pack2(sc[c * 32 + i], sc[c * 32 + i + 1]), s2, nm2), e0, e1);
            e0 = fast_exp2(e0);
            e1 = fast_exp2(e1);
            pk[i >> 1] = pack_bf16x2(e0, e1);
            sums[(i >> 1) & 1] = add2(sums[(i >> 1) & 1], pack2(e0, e1));
          }
          if (C::P_APART && c == 0) wait(&pv_done[x], ph ^ 1u);  // the P before this one
          tmem_st_32x16(p_col + c * 16, pk);
        }
        float sum0, sum1;
        unpack2(add2(sums[0], sums[1]), sum0, sum1);
        l += sum0 + sum1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
        ph ^= 1u;
      }
      passed += (uint32_t)(w.end - w.begin);
      const bool starts = w.begin == 0, ends = w.end == w.units;
      const long long slot = 2 * (long long)blockIdx.x + (starts ? 1 : 0);
      const long long part = slot * (2 * kBM) + x * kBM;
      if (end > w.begin) {
        // normalise and write out, or leave the part for the join.  The next item's first product overwrites O only after
        // these warps delivered its P.
        wait(&pv_done[x], ph ^ 1u);
        tc_fence_after();
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        const float inv = 1.f / l;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 64) {  // all loads of 64 columns first: they take as long as one
          float v[2][2][16];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              tmem_ld_16x256b_x4(tmem_base + o_col + ((uint32_t)(quad * 32 + hh * 16) << 16) + c0 + c * 32, v[hh][c]);
          tmem_ld_wait();
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // rows lane >> 2 and that + 8
              const int r = hh * 16 + half * 8 + (lane >> 2);
              const float f = __shfl_sync(0xffffffffu, inv, r);
              int token, h;
              const bool there = row_of(p, tl, w.n, w.head, w.item, x, quad * 32 + r, token, h);
              if (starts && ends) {
                bf16* dst = p.out + ((long long)(w.first + token) * p.heads + h) * D + c0 + (lane & 3) * 8;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  uint32_t t[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) t[k] = pack_bf16x2(v[hh][c][4 * k + 2 * half] * f, v[hh][c][4 * k + 2 * half + 1] * f);
                  quad_transpose(t, lane);
                  if (there) *reinterpret_cast<uint4*>(dst + c * 32) = make_uint4(t[0], t[1], t[2], t[3]);
                }
              } else if (there) {
                float* dst = parts.acc + (part + quad * 32 + r) * D + c0 + (lane & 3) * 2;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float2*>(dst + c * 32 + k * 8) = make_float2(v[hh][c][4 * k + 2 * half], v[hh][c][4 * k + 2 * half + 1]);
              }
            }
        }
      }
      if (!(starts && ends)) parts.ml[part + row_in_tile] = make_float2(m_used, l);
      if (starts && !ends) share.b = w.b, share.head = w.head, share.item = w.item;
      if (first_item) share.continues = !starts, share.ends = ends;
      first_item = false;
    }
    if (threadIdx.x == 128) parts.share[blockIdx.x] = share;
    if (share.continues < 0) parts.ml[2ll * blockIdx.x * (2 * kBM) + x * kBM + row_in_tile] = make_float2(-INFINITY, 0.f);
    if (*abort_flag != 0 && lane == 0) atomicCAS(p.status, 0, kStatusEpilogueTimeout);
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // a wait gave up: let copies that are still in flight land before the CTA retires
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
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

// [tokens][heads][head_dim] of the queries; box = 64 columns of a query tile's heads and tokens
bool queries_tmap(CUtensorMap* map, const PagedAttention& p, int head_dim, const Tiling& tl) {
  EncodeFn fn = attn_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)p.heads, (cuuint64_t)p.tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)(p.heads == 1 ? head_dim : p.q_head) * 2, (cuuint64_t)(p.tokens == 1 ? head_dim : p.q_token) * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)tl.group, (cuuint32_t)(tl.tokens / tl.tiles)}, estr[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(p.q), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT && bind_primary_context()) r = encode();  // the first call of a thread
  return r == CUDA_SUCCESS;
}

// How a call is run.  Either kernel takes any rows; what a sequence typically has decides: twice the mean, or the most where the
// caller knows less.
struct Plan {
  Tiling tl;
  bool many = false;  // rows for the tcgen05 kernel
  int ctas, cluster = 0, items = 0;  // cluster > 0: CTAs of an item, and the items that a sequence and head can have
  Plan(const PagedAttention& p, int head_dim) {
    const long long group = p.heads / p.kv_heads, typical = std::min<long long>(p.max_new, (2ll * p.tokens + p.seqs - 1) / p.seqs);
    const long long rows = typical * group, keys = (long long)p.max_pages << p.page_shift;
    const int sms = attn_grid(1 << 20);
    if (group <= 64) {
      tl = Tiling(p, rows <= 16 ? 16 : rows <= 32 ? 32 : 64, 1, kRowsFixed);
      // An item per cluster, without a second kernel, where the keys of its CTAs are few even if a sequence fills its row of the
      // page table, which is all that the host knows: at most 4096 each, or 1024 where the clusters leave half of the SMs idle.  Both ways
      // (us, shares / clusters; 32 heads on 8 of 128): one token over 1000 keys 12.0 / 6.9, over 4000 13.7 / 9.0, over 16000 17.5 / 20.5;
      // 8 of 8000 52.0 / 44.7, 32 of up to 4000 54.2 / 48.2, 64 of 1000 54.7 / 46.0, 64 of 4000 165.7 / 149.5; of 8000 keys a CTA 40 items
      // 201 / 227, which the limit of 4096 is for, 64 of up to 8000, where clusters would be the better ones, 138 / 131.
      const long long most = (p.max_new + tl.per - 1) / tl.per, all = (long long)p.seqs * tl.heads * most;
      const long long slots = (long long)sms * (head_dim == 64 && tl.height < 64 ? 3 : 2);
      const long long likely = (long long)p.seqs * tl.heads * ((typical + tl.per - 1) / tl.per);
      // More rows are better off there too while there is little work, at most 40 (20 of heads of 128) blocks of 64 rows by 64 keys per
      // SM.  tcgen05 kernel / clusters (us): 12 heads of 64, 1 x 100 tokens 14.8 / 9.2, 4 x 300 24.8 / 9.3 (8 blocks), 8 x 500 32.6 / 26.6
      // (41), 24 x 200 after 500 47.2 / 57.7 (86); 32 heads on 8 of 128, 1 x 400 25.2 / 14.8 (9.5), 1 x 700 34.3 / 26.6 (26), 1 x 200 after
      // 3000 40.7 / 52.8 (35).
      if (rows <= 64 || likely * ((keys + kKeys - 1) / kKeys) <= sms * 2560ll / head_dim) {
        for (int c = kFewCluster; c >= 1; c /= 2) {
          if (c > 1 ? all * c > slots || keys <= c * (kKeys / 2) : all > kFewItems) continue;
          if (keys <= c * (2 * all * c < slots ? 1024ll : 4096ll)) {
            cluster = c;
            items = (int)most;
            ctas = (int)all * c;
          }
          break;
        }
      }
    }
    if (cluster == 0 && rows > 64) {
      many = true;
      tl = Tiling(p, kBM, 2, kChunkFixed);
    }
    if (cluster == 0) {
      ctas = sms * (many ? 1 : 2);
      for (int h = 1; h <= tl.heads && h <= ctas; ++h)
        if (tl.heads % h == 0 && ctas % h == 0) tl.side = h;
    }
  }
  int rows() const { return tl.height * tl.tiles; }
};

template <typename C>
cudaError_t rows_launch(const PagedAttention& p, const Parts& parts, const Plan& plan, cudaStream_t stream) {
  CUtensorMap tk, tv;
  const int box = std::min(kKeys, 1 << p.page_shift);
  if (!pages_tmap(&tk, p.k_pages, p, C::D, p.k_page, p.k_row, p.k_head, box) || !pages_tmap(&tv, p.v_pages, p, C::D, p.v_page, p.v_row, p.v_head, box))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> granted{0};
  const cudaError_t e = once_per_device(granted, [] {
    return cudaFuncSetAttribute(paged_rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_rows_kernel<C>, dim3(plan.ctas), dim3(kRowsThreads), C::SMEM, stream, C::FEW && plan.cluster > 1 ? plan.cluster : 0, tk, tv,
                    p, parts, plan.tl);
}
template <int D, bool FEW>
cudaError_t rows_launch_d(const PagedAttention& p, const Parts& parts, const Plan& plan, cudaStream_t stream) {
  return plan.rows() == 16   ? rows_launch<Rows<D, 1, FEW>>(p, parts, plan, stream)
         : plan.rows() == 32 ? rows_launch<Rows<D, 2, FEW>>(p, parts, plan, stream)
                             : rows_launch<Rows<D, 4, FEW>>(p, parts, plan, stream);
}

template <int D>
cudaError_t chunk_launch(const PagedAttention& p, const Parts& parts, const Plan& plan, cudaStream_t stream) {
  using C = Chunk<D>;
  CUtensorMap tq, tk, tv;
  const int box = std::min(kBM, 1 << p.page_shift);
  if (!queries_tmap(&tq, p, D, plan.tl) || !pages_tmap(&tk, p.k_pages, p, D, p.k_page, p.k_row, p.k_head, box) ||
      !pages_tmap(&tv, p.v_pages, p, D, p.v_page, p.v_row, p.v_head, box))
    return cudaErrorInvalidValue;
  auto kernel = paged_chunk_kernel<D>;
  static std::atomic<unsigned long long> granted{0};
  const cudaError_t e = once_per_device(granted, [&] {
    cudaFuncAttributes fa;
    // the register shares of the kernel's warps add up to what it is launched with, or the larger one waits forever
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs != 168) return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(plan.ctas), dim3(kChunkThreads), C::SMEM, stream, 0, tq, tk, tv, p, parts, plan.tl);
}

template <int D>
cudaError_t attention_launch(const PagedAttention& p, void* work, int* launches, cudaStream_t stream) {
  const Plan plan(p, D);
  *launches = plan.cluster > 0 ? 1 : 2;
  Parts parts{};
  if (plan.cluster > 0) {
    parts.cluster = plan.cluster;
    parts.items = plan.items;
    return rows_launch_d<D, true>(p, parts, plan, stream);
  }
  parts.acc = reinterpret_cast<float*>(work);
  parts.ml = reinterpret_cast<float2*>(parts.acc + 2ll * plan.ctas * plan.rows() * D);
  parts.share = reinterpret_cast<Share*>(parts.ml + 2ll * plan.ctas * plan.rows());
  const cudaError_t e = !plan.many ? rows_launch_d<D, false>(p, parts, plan, stream) : chunk_launch<D>(p, parts, plan, stream);
  if (e != cudaSuccess) return e;
  // of a tile's rows those that a sequence can have
  const long long most = std::min<long long>(plan.rows(), (long long)p.max_new * (p.heads / p.kv_heads));
  if (!plan.many)
    return launch_pdl(paged_join_kernel<D, 4>, dim3(plan.ctas, (unsigned)std::min<long long>(most, 16)), dim3(128), 0, stream, 0, p, parts, plan.tl);
  return launch_pdl(paged_join_many_kernel<D>, dim3(plan.ctas, plan.rows() / (kJoinWarps * kJoinRows)), dim3(32 * kJoinWarps), 0, stream, 0, p, parts,
                    plan.tl);
}

}  // namespace

long long paged_attention_workspace(const PagedAttention& p, int head_dim) {
  const Plan plan(p, head_dim);
  if (plan.cluster > 0) return 0;
  return 2ll * plan.ctas * plan.rows() * (head_dim * sizeof(float) + sizeof(float2)) + plan.ctas * sizeof(Share);
}

cudaError_t paged_attention_launch(const PagedAttention& p, int head_dim, void* work, int* launches, cudaStream_t stream) {
  if (head_dim == 64) return attention_launch<64>(p, work, launches, stream);
  if (head_dim == 128) return attention_launch<128>(p, work, launches, stream);
  return cudaErrorInvalidValue;
}

}  // namespace dion
