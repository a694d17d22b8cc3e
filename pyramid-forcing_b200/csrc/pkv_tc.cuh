// Blackwell tensor-core building blocks shared by the attention kernels: PTX
// wrappers (mbarrier, TMA, tcgen05), bounded waits, paired fp32 arithmetic, the
// per-row softmax of a 128 x 128 score tile, and the host side of tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "pkv_common.cuh"
#include "pkv_f2.cuh"

namespace pkv {

constexpr int kBM = 128;          // query rows per tile (= TMEM lanes)
constexpr int kBN = 128;          // keys per tile
constexpr int kHD = 128;          // head dim of the tensor-core path
constexpr uint32_t kHalfBytes = kBM * 64 * 2;   // [128 rows][64 bf16] = 16 KB
constexpr uint32_t kTileBytes = 2 * kHalfBytes; // one 128x128 bf16 tile
constexpr uint64_t kTimeoutNs = 4000000000ull;  // 4 s per wait
constexpr float kRescaleThreshold = 8.0f;        // log2 units

// ---- PTX wrappers -----------------------------------------------------------
__device__ __forceinline__ uint32_t su32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(su32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait: false when the CTA is aborting (limit reached here or in
// another role).
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort,
                                          int32_t* status, uint64_t limit_ns = kTimeoutNs) {
  if (mbar_try(b, parity)) return true;
  const uint64_t t0 = now_ns();
  while (!mbar_try(b, parity)) {
    if (*abort) return false;
    if (now_ns() - t0 > limit_ns) {
      *abort = 1;
      flag(status, PKV_ST_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(su32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(su32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(su32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(su32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Pull a tile of a tensor into L2 ahead of its load (no shared memory, no
// completion to wait for).
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// True in one lane of a converged warp.  MMAs issued behind it are issued faster
// than behind a comparison of lane numbers: 48 cycles instead of 55 to 66 for one
// of M = 128, N = 64, K = 16.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          su32(bar))
      : "memory");
}
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// 32 consecutive TMEM columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Larger of two, NaN if either is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x for a pair (x <= 126), on the FMA pipe: Cody-Waite reduction x = n + f with
// n = rint(x) (the addend of 1.5 * 2^23, and 128 for an exponent field, leaves
// n + 128 in the low mantissa bits) and f in [-0.5, 0.5], half a cubic for 2^f,
// times 2^(n + 1).  Cubic coefficients: minimax relative-error fit of 2^f on
// [-0.5, 0.5] (exp2_poly_fit.py beside this file), max relative error 7.5e-5 -- far
// below the 2^-8 step of the bf16 P it produces.  x is clamped at -128, whose field
// is 0: anything from there down, -inf too, gives 0, and NaN stays NaN.
__device__ __forceinline__ f2 exp2_poly2(f2 x) {
  constexpr float kRound = 12582912.0f + 128.0f;  // 1.5 * 2^23 + 128
  float x0, x1;
  un2(x, x0, x1);
  x = mk2(max_nan(x0, -128.0f), max_nan(x1, -128.0f));
  const f2 rnd = mk2(kRound, kRound);
  const f2 t = add2(x, rnd);                            // n + 128 in the low bits of t
  const f2 f = sub2(x, sub2(t, rnd));                   // f = x - n
  auto half2 = [](float c) { return mk2(0.5f * c, 0.5f * c); };
  f2 p = fma2(half2(0.0551716685295105f), f, half2(0.2426111251115799f));
  p = fma2(p, f, half2(0.6932609677314758f));
  p = fma2(p, f, half2(0.9999280571937561f));
  float t0, t1;
  un2(t, t0, t1);
  // t's bit pattern is 0x4B400000 + n + 128; shifted left by 23 it is 2^(n + 1)
  return mul2(p, mk2(__uint_as_float(__float_as_uint(t0) << 23),
                     __uint_as_float(__float_as_uint(t1) << 23)));
}

// UMMA shared-memory descriptor, 128-byte swizzle (SM100 version bits = 1).
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= uint64_t((saddr >> 4) & 0x3FFFu);
  d |= uint64_t((lbo >> 4) & 0x3FFFu) << 16;
  d |= uint64_t((sbo >> 4) & 0x3FFFu) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
// Instruction descriptor, kind::f16: bf16 A/B, fp32 D, M=128, N=128.
__host__ __device__ constexpr uint32_t idesc_bf16(bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_mn_major) << 16) |
         (uint32_t(kBN >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
}

// Row max over 128 raw scores held as bits (tree of 3-input max).
__device__ __forceinline__ float row_max128(const uint32_t (&s)[4][32]) {
  float m[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float a[11];
#pragma unroll
    for (int i = 0; i < 10; ++i)
      a[i] = max3(__uint_as_float(s[q][3 * i]), __uint_as_float(s[q][3 * i + 1]),
                  __uint_as_float(s[q][3 * i + 2]));
    a[10] = fmaxf(__uint_as_float(s[q][30]), __uint_as_float(s[q][31]));
    const float b0 = max3(a[0], a[1], a[2]), b1 = max3(a[3], a[4], a[5]);
    const float b2 = max3(a[6], a[7], a[8]), b3 = fmaxf(a[9], a[10]);
    m[q] = fmaxf(max3(b0, b1, b2), b3);
  }
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// Which column pairs of a 32-column chunk take the FMA-pipe exp2: 3 of 16
// (pairs 2, 7, 12).  Measured on B200 (attention kernel case, one call):
// 0.5245 ms with 3 of 16, 0.5263 with 4, 0.5284 with 2, 0.543 with 6, 0.567
// with 8, and all on MUFU 1.4% slower than 6 of 16: the FMA / ALU side is
// the more contended pipe.
__host__ __device__ constexpr bool poly_pair(int i) { return i % 5 == 2; }

// P for 32 columns (16 pairs) of one row: p = 2^(s * scale - m), summed into
// two paired accumulators and packed to bf16 pairs.
template <bool kMixed>
__device__ __forceinline__ void softmax_chunk(const uint32_t (&s)[32], f2 scale2, f2 negm2,
                                              f2& acc0, f2& acc1, uint32_t (&pr)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const f2 x = fma2(mk2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2,
                      negm2);
    f2 p;
    if (kMixed && poly_pair(i)) {
      p = exp2_poly2(x);
    } else {
      float x0, x1;
      un2(x, x0, x1);
      p = mk2(fast_exp2(x0), fast_exp2(x1));
    }
    if (i & 1)
      acc1 = add2(acc1, p);
    else
      acc0 = add2(acc0, p);
    float p0, p1;
    un2(p, p0, p1);
    pr[i] = pack_bf16x2(p0, p1);
  }
}

// Store one warp's 32 rows x 128 columns of fp32 as normalised bf16 rows.
__device__ __forceinline__ void store_row32(uint16_t* dst, const uint32_t (&o)[32], float inv) {
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    uint4 w;
    w.x = pack_bf16x2(__uint_as_float(o[e + 0]) * inv, __uint_as_float(o[e + 1]) * inv);
    w.y = pack_bf16x2(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
    w.z = pack_bf16x2(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
    w.w = pack_bf16x2(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
    *reinterpret_cast<uint4*>(dst + e) = w;
  }
}

// ---- host side ----------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

inline bool make_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims,
                     const cuuint64_t* strides_bytes, const cuuint32_t* box) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims,
                        strides_bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

}  // namespace pkv
