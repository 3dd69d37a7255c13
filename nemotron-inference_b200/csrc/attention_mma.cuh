// What the attention kernels share: tensor-core instructions on 16- and 8-bit operands, wider TMEM
// accesses, and the exponential.
#pragma once

#include "common.cuh"

namespace nmoe {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Instruction descriptor of kind::f16 on bf16 operands, FP32 sums, M = 128.  `b_rows_along_n`: B lies
// in shared memory as rows of consecutive n (values: a token's row), not of consecutive k.
__host__ __device__ constexpr uint32_t make_idesc_bf16(uint32_t n, bool b_rows_along_n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_rows_along_n ? 1u << 16 : 0u) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}

// D[tmem] (+)= A[smem] B[smem]^T
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// D[tmem] (+)= A[tmem] B[smem]^T
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// 32 consecutive columns of this warp's 32 lanes, without the wait (see tmem_ld_x16_async).
__device__ __forceinline__ void tmem_ld_x32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

template <int N>
__device__ __forceinline__ void registers_loaded(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x for two x <= 120 without the unit for special functions, which takes sixteen a cycle on an SM: x is split
// into the nearest whole number and a rest f, 2^f is a polynomial 1 + f (c1 + f (c2 + ...)) whose largest
// relative error over |f| <= 1/2 is as small as the leading 1 allows (1.0e-4 of degree 3, 2.9e-6 of degree 4),
// and the power of two of the whole number multiplies it.  0 for x <= -127, NaN for NaN.
template <int Degree>
__device__ __forceinline__ uint64_t exp2_polynomial2(uint64_t x) {
  static_assert(Degree == 3 || Degree == 4);
  constexpr float kToWhole = 12582912.0f;  // 1.5 * 2^23: the sum's last bits are the nearest whole number
  float x0, x1;
  unpack2(x, x0, x1);
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x0));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x1));
  x = pack2(x0, x1);
  const uint64_t whole = add2(x, pack2(kToWhole, kToWhole));
  const uint64_t f = fma2(add2(whole, pack2(-kToWhole, -kToWhole)), pack2(-1.0f, -1.0f), x);
  uint64_t p;
  if constexpr (Degree == 3) {
    p = fma2(pack2(0.055009060f, 0.055009060f), f, pack2(0.24221097f, 0.24221097f));
    p = fma2(p, f, pack2(0.69328290f, 0.69328290f));
  } else {
    p = fma2(pack2(0.0095825763f, 0.0095825763f), f, pack2(0.055906828f, 0.055906828f));
    p = fma2(p, f, pack2(0.24024107f, 0.24024107f));
    p = fma2(p, f, pack2(0.69312412f, 0.69312412f));
  }
  p = fma2(p, f, pack2(1.0f, 1.0f));
  float w0, w1;
  unpack2(whole, w0, w1);
  return mul2(p, pack2(__uint_as_float((__float_as_uint(w0) << 23) + 0x3f800000u),
                       __uint_as_float((__float_as_uint(w1) << 23) + 0x3f800000u)));
}

// Two values as bf16, `lo` in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}

// A sector of a row, from a 16-byte boundary; in one piece where that is one of 32.
__device__ __forceinline__ void store_32_bytes(void* to, const uint32_t (&w)[8], bool aligned) {
  if (aligned) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Registers of four warps, all of which call it: what some give up others take, out of those that the
// block was launched with.
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// The bounded wait of mbar_wait_warp(), without a call: a function's registers are not known to the
// split above.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) {
  bool done = mbar_try_wait_at(bar, parity);
  if (__all_sync(0xffffffffu, done)) return true;
  const long long start = clock64();
  while (!done && clock64() - start < (1ll << 31)) done = mbar_try_wait_at(bar, parity);
  return __all_sync(0xffffffffu, done);
}

// Asks for the next block of the grid that has not begun, in place of its launch; 16 bytes arrive on
// the barrier.  After an answer that there is none, it is not asked again.
__device__ __forceinline__ void request_next_block(uint32_t answer, uint32_t bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
      ::"r"(answer), "r"(bar)
      : "memory");
}
// The block's index, -1 for none.
__device__ __forceinline__ int next_block(uint32_t answer) {
  int block;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "mov.b32 %0, -1;\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, r;\n\t}"
      : "=r"(block)
      : "r"(answer)
      : "memory");
  return block;
}

}  // namespace nmoe
