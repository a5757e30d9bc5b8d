// Inline-PTX wrappers used by the attention kernels beside those of ptx.cuh:
// four-dimensional TMA loads, tensor-core products whose A operand lies in
// TMEM, TMEM stores, and 2^x.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace bdion {

// Status codes of the attention kernels' bounded waits (see common.cuh).
constexpr int kStatusWindowProducerTimeout = 0x401;
constexpr int kStatusWindowMmaTimeout = 0x402;
constexpr int kStatusWindowSoftmaxTimeout = 0x403;

__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Untiled copy of `bytes` (a multiple of 16, both addresses 16-byte aligned).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Shared-memory operands of the 128-byte swizzle by the low word of their
// descriptor (make_sdesc_sw128: address and leading-dimension offset); the high
// word (8-row stride 1024, version, layout) is the same for all of them.
constexpr uint32_t kSdescHigh = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ constexpr uint32_t sdesc_low(uint32_t saddr, uint32_t lbo) {
  return (saddr >> 4) | ((lbo >> 4) << 16);
}

// tcgen05.mma issued by the one lane whose `leader` is set, without a branch: in
// code that one lane has branched into, the operands took their own way to
// uniform registers and every product some 90 cycles to issue.
//   umma_ss: D[tmem] (+)= A[smem] * B[smem]^T
//   umma_ts: D[tmem] (+)= A[tmem] * B[smem]^T, A as packed 16-bit pairs, one per 32-bit column
__device__ __forceinline__ void umma_ss(bool leader, uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                        bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred P, Q;\n"
      ".reg .b64 A, B;\n"
      "setp.ne.b32 P, %4, 0;\n"
      "setp.ne.b32 Q, %5, 0;\n"
      "mov.b64 A, {%1, %6};\n"
      "mov.b64 B, {%2, %6};\n"
      "@Q tcgen05.mma.cta_group::1.kind::f16 [%0], A, B, %3, P;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"((uint32_t)accumulate), "r"((uint32_t)leader), "n"(kSdescHigh)
      : "memory");
}
__device__ __forceinline__ void umma_ts(bool leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc,
                                        bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred P, Q;\n"
      ".reg .b64 B;\n"
      "setp.ne.b32 P, %4, 0;\n"
      "setp.ne.b32 Q, %5, 0;\n"
      "mov.b64 B, {%2, %6};\n"
      "@Q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], B, %3, P;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"((uint32_t)accumulate), "r"((uint32_t)leader), "n"(kSdescHigh)
      : "memory");
}
// Arrive on `bar` once every product that this lane has issued is done.
__device__ __forceinline__ void umma_commit_by(bool leader, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred Q;\n"
      "setp.ne.b32 Q, %1, 0;\n"
      "@Q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar)),
      "r"((uint32_t)leader)
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// thread t writes lane (base + t), columns col .. col + 31
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t* r) {
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
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of floats: one instruction works on both.
using f2 = unsigned long long;
__device__ __forceinline__ f2 make_f2(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float lo_of(f2 x) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
  return lo;
}
__device__ __forceinline__ float hi_of(f2 x) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
  return hi;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// the larger of two, NaN where one of them is (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of a pair on the FMA pipes: x = n + f with n the nearest whole number (by
// adding 1.5 * 2^23, whose low bits then hold n) and f in [-1/2, 1/2]; 2^f by a
// polynomial of degree 4 (minimax in relative error, found by reweighted least
// squares with the constant term held at 1: off by 2^-18.4 at most), times 2^n,
// whose bits are n + 127 in the exponent's place. x is at most 127; from -127 down
// the result is exactly 0 (the exponent's place is 0). A NaN stays one: it goes
// through the polynomial, and the product keeps it whatever 2^n becomes.
__device__ __forceinline__ f2 ex2_poly(f2 x) {
  x = make_f2(max_nan(lo_of(x), -127.f), max_nan(hi_of(x), -127.f));
  const f2 t = add2(x, make_f2(12582912.f, 12582912.f));
  const f2 n = add2(t, make_f2(-12582912.f, -12582912.f));
  const f2 f = fma2(n, make_f2(-1.f, -1.f), x);
  f2 p = fma2(f, make_f2(0.009582853f, 0.009582853f), make_f2(0.055906426f, 0.055906426f));
  p = fma2(p, f, make_f2(0.24024099f, 0.24024099f));
  p = fma2(p, f, make_f2(0.69312418f, 0.69312418f));
  p = fma2(p, f, make_f2(1.f, 1.f));
  return mul2(p, make_f2(__uint_as_float((__float_as_uint(lo_of(t)) << 23) + 0x3f800000u),
                         __uint_as_float((__float_as_uint(hi_of(t)) << 23) + 0x3f800000u)));
}
// 2^x of pair `i` of a row: one pair in kPolyEvery by the polynomial, the others by the
// special-function unit, whose four results a cycle and quarter of an SM bound these
// kernels otherwise.
constexpr int kPolyEvery = 4;
__device__ __forceinline__ f2 ex2_pair(int i, f2 x) {
  return i % kPolyEvery == kPolyEvery - 1 ? ex2_poly(x) : make_f2(ex2(lo_of(x)), ex2(hi_of(x)));
}

// two floats as a packed pair of the element type, `lo` in the low half
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(f2 x, T tag) {
  return pack2(lo_of(x), hi_of(x), tag);
}

}  // namespace bdion
