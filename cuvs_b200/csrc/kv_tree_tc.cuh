// The tensor-core kernel's PTX and shape: what kv_tree_tc.cu has beside tc_ptx.cuh.
#pragma once

#include "kv_tree.cuh"
#include "tc_ptx.cuh"

namespace cuvs_b200::kv {

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
  asm volatile(
    "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
    "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
    "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
    "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
    : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A step of 16 keys: weights [128 rows x 16 keys] from tensor memory, and values by the low word of the descriptor of a tile whose rows are the
// product's depth: 64 columns of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes apart; bits 16 on of the word: the way to the next 64 columns.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t lo_b, uint32_t idesc, bool add)
{
  constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
  asm volatile(
    "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
    "setp.ne.b32 p, %5, 0;\n\t"
    "mov.b64 b, {%2, %4};\n\t"
    "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
    ::"r"(tmem_d), "r"(tmem_a), "r"(lo_b), "r"(idesc), "r"(kHi), "r"(uint32_t(add))
    : "memory");
}

template <int N>
__device__ __forceinline__ void registers_up()
{
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down()
{
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A weight of 32 bits as the sum of two 16-bit numbers, so that a row of the output is off by little more than its own rounding: what one number
// loses (2^-9 of each weight in bf16, 2^-12 in fp16) is as much as that.  Neither number is 0 where the weight is 2^-30 of the largest or more: 0 times an
// infinite value would be no number.
// kAhead: by how much (as a power of two) a running top may be behind before sums are brought back to it.
constexpr float kAhead = 4.0f;
template <typename T>
struct weight_pair;
template <>
struct weight_pair<__half> {
  // 11 bits, cut off, and the rest rounded to 11 bits.  Weights are held times 2^11 (and up to 2^4 more: below fp16's 65,504), so that small ones keep
  // their digits above fp16's smallest number, 2^-24: it is 2^-35 of the largest weight, or 2^-31 where the top is behind.
  static __device__ __forceinline__ void split(float a, float b, uint32_t& high, uint32_t& low)
  {
    // Of a little less than the weight, by a step of 32 bits and fp16's smallest number: the rest is not rounded to 0.  (Less than 0 is cut off to 0.)
    constexpr float kLess = 1.0f - 1.1920928955078125e-7f, kSmallest = 5.9604644775390625e-8f;  // 1 - 2^-23, 2^-24
    float x, y, u, v;
    fma2(two(a, b), two(kLess, kLess), two(-kSmallest, -kSmallest)).get(x, y);
    asm("cvt.rz.relu.f16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(y), "f"(x));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&high));
    add2(two(a, b), two(-h.x, -h.y)).get(u, v);
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(low) : "f"(u), "f"(v));
  }
  static __device__ __forceinline__ float2 join(uint32_t high, uint32_t low)
  {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&high)), b = __half22float2(*reinterpret_cast<const __half2*>(&low));
    return make_float2(a.x + b.x, a.y + b.y);
  }
};
template <>
struct weight_pair<__nv_bfloat16> {
  // 8 bits, cut off, and the rest rounded to 8 bits: to 2^-17 of the weight.  (The rest comes times 1 + 2^-22 of the weight: more than nothing.)
  static __device__ __forceinline__ void split(float a, float b, uint32_t& high, uint32_t& low)
  {
    constexpr float kMore = 1.0f + 2.384185791015625e-7f;
    high = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    const float x = __uint_as_float(__float_as_uint(a) & 0xFFFF0000u), y = __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
    float u, v;
    fma2(two(a, b), two(kMore, kMore), two(-x, -y)).get(u, v);
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(low) : "f"(u), "f"(v));
  }
  static __device__ __forceinline__ float2 join(uint32_t high, uint32_t low)
  {
    return make_float2(__uint_as_float(high << 16) + __uint_as_float(low << 16), __uint_as_float(high & 0xFFFF0000u) + __uint_as_float(low & 0xFFFF0000u));
  }
};

// cap tanh(y) for scores that are capped: below kTanhNear y times a polynomial of y^2 (tree_view::cap_near), else by an exponential (to 2^-22).
__device__ __forceinline__ two tanh_near(two y, const float (&c)[5])
{
  const two z = mul2(y, y);
  two p       = fma2(z, two(c[4], c[4]), two(c[3], c[3]));
  p           = fma2(z, p, two(c[2], c[2]));
  p           = fma2(z, p, two(c[1], c[1]));
  p           = fma2(z, p, two(c[0], c[0]));
  return mul2(y, p);
}
__device__ __forceinline__ float tanh_far(float y)
{
  const float e = power_of_2(2.8853900817779268f * fabsf(y));  // 2 log2(e)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
  return copysignf(fmaf(-2.0f, r, 1.0f), y);
}

}  // namespace cuvs_b200::kv
