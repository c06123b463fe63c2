// Building blocks of the attention kernels (attention.cu, paged_attention.cu): products with descriptors stepped by one addition,
// two fp32 operations per instruction, tensor-memory copies, division by multiplication, register shares.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

#include "gemm.h"
#include "umma.cuh"

namespace dion {

namespace {

constexpr int kBM = 128;  // rows of a tile, of queries and of keys
constexpr float kRescaleThreshold = 8.f;  // log2 units

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const float (&v)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The MMA-issuing thread is on the critical path of every kv iteration (tiles are small, so one
// tcgen05.mma runs for only 30-70 cycles); descriptors are therefore kept as two 32-bit halves and
// stepped with a single integer add: the start-address field (bits [0,14), units of 16 bytes) never
// carries because shared-memory offsets stay below 256 KB.
struct DescHalves {
  uint32_t lo, hi;
};
__device__ __forceinline__ DescHalves desc_halves(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  const uint64_t d = make_smem_desc(smem_addr, lbo_bytes, sbo_bytes);
  return DescHalves{(uint32_t)d, (uint32_t)(d >> 32)};
}
// D[tmem] (+)= A[smem] * B[smem], bf16, descriptors given as halves plus byte offsets
__device__ __forceinline__ void umma_ss_h(uint32_t tmem_d, DescHalves a, uint32_t a_off, DescHalves b, uint32_t b_off,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(tmem_d),
      "r"(a.lo + (a_off >> 4)), "r"(a.hi), "r"(b.lo + (b_off >> 4)), "r"(b.hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_ts_h(uint32_t tmem_d, uint32_t tmem_a, DescHalves b, uint32_t b_off,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b.lo + (b_off >> 4)), "r"(b.hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.  The softmax loops issue 7 to 14 instructions per score without them and are
// what the tensor core waits for; with them 3 to 5, of which one is the exponential.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  const __nv_bfloat162 h2 = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h2);
}

// untiled bulk copy global -> shared (both 16-byte aligned, size a multiple of 16), completing on `bar`
__device__ __forceinline__ void bulk_load_1d(void* smem_dst, const void* gsrc, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(gsrc), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994); the integer division of the device takes some
// hundred cycles, and a role does several of them before it can start on a tile
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(int divisor) : d((uint32_t)divisor), m(0), s(0) {
    while (s < 31 && (1u << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s); }
};

// Position in a ring of N stages and the parity of the barrier phase that fills it next
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1u;
    }
  }
};

// 16 lanes x 32 fp32 columns: lane t receives, for k = 0..3, columns 8k + 2 (t & 3) and + 1 of row t >> 2 (v[4k], v[4k + 1])
// and of row (t >> 2) + 8 (v[4k + 2], v[4k + 3])
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 128 rows x 32 bytes from shared memory (a K-major operand tile) to 8 columns of tensor memory
__device__ __forceinline__ void tmem_cp_128x32b(uint32_t taddr, DescHalves d, uint32_t off) {
  asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.128x256b [%0], d;\n\t}" ::"r"(taddr),
               "r"(d.lo + (off >> 4)), "r"(d.hi)
               : "memory");
}
// v[k] of lane q of each group of four becomes v[q] of lane k
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[4], int lane) {
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1) {
    const bool up = lane & b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & b) continue;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i | b], b);
      if (up) v[i] = got;
      else v[i | b] = got;
    }
  }
}
// D[128 x 128] = A B^T over the head dimension, both K-major tiles; A from tensor memory (a_col) where kTmemA
template <int D, bool kTmemA>
__device__ __forceinline__ void scores(uint32_t d_col, DescHalves a, uint32_t a_col, DescHalves b, uint32_t b_off) {
  constexpr uint32_t idesc = make_instr_desc(1, kMajorK, kMajorK, kBM, kBM);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = (kk >> 2) * (kBM * 128) + (kk & 3) * 32;
    if constexpr (kTmemA) umma_ts_h(d_col, a_col + kk * 8, b, b_off + off, idesc, kk > 0 ? 1u : 0u);
    else umma_ss_h(d_col, a, off, b, b_off + off, idesc, kk > 0 ? 1u : 0u);
  }
}
// Register shares of the first warpgroup and of the eight softmax warps after it: together no more than the 384 x 168 that
// the launch has, or the larger share waits forever
template <int kFirst, int kSoftmax>
__device__ __forceinline__ void give_registers() {
  static_assert(128 * kFirst + 256 * kSoftmax <= 384 * 168 && kFirst % 8 == 0 && kSoftmax % 8 == 0);
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFirst));
}
template <int kFirst, int kSoftmax>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmax));
}
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn attn_encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(sym);
  });
  return fn;
}

// CTAs of a persistent kernel with one CTA per SM
int attn_grid(long long items) {
  static std::atomic<int> known[64];  // per device; the count does not change
  int dev = 0;
  cudaGetDevice(&dev);
  int sms = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  }
  return (int)(items < sms ? items : sms);
}

}  // namespace

}  // namespace dion
