// The tensor-core kernel's PTX and shape: what kv_tree_tc.cu has beside tc_ptx.cuh.
#pragma once

#include "kv_tree.cuh"
#include "tc_ptx.cuh"

namespace cuvs_b200::kv {

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]));
  asm volatile("" : "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
               "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A row-block of weights in tensor memory times values: A [128 rows x 16 keys] from tensor memory.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate)
{
  asm volatile(
    "{\n\t.reg .pred p;\n\t"
    "setp.ne.b32 p, %4, 0;\n\t"
    "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
    ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
    : "memory");
}

// Shared-memory descriptor of a tile whose rows are the product's depth (keys): 64 columns of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes apart,
// the next 64 columns `panel` bytes on.
__device__ __forceinline__ uint64_t make_desc_sw128_rows(uint32_t saddr, uint32_t panel)
{
  uint64_t d = 0;
  d |= uint64_t((saddr & 0x3FFFFu) >> 4);
  d |= uint64_t(panel >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
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
// loses (2^-9 of each weight in bf16, 2^-12 in fp16) is as much as that.  The second number is never 0 where the first is not: 0 times an infinite value
// would be no number.
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
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(high) : "f"(b), "f"(a));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&high));
    const __half2 rest = __floats2half2_rn(a - h.x, b - h.y);
    low                = __vmaxu2(*reinterpret_cast<const uint32_t*>(&rest), __vminu2(high, 0x00010001u));
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
    high                   = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    const float x          = fmaf(a, 1.0f + 2.384185791015625e-7f, -__uint_as_float(__float_as_uint(a) & 0xFFFF0000u));
    const float y          = fmaf(b, 1.0f + 2.384185791015625e-7f, -__uint_as_float(__float_as_uint(b) & 0xFFFF0000u));
    const __nv_bfloat162 l = __floats2bfloat162_rn(x, y);
    low                    = *reinterpret_cast<const uint32_t*>(&l);
  }
  static __device__ __forceinline__ float2 join(uint32_t high, uint32_t low)
  {
    return make_float2(__uint_as_float(high << 16) + __uint_as_float(low << 16), __uint_as_float(high & 0xFFFF0000u) + __uint_as_float(low & 0xFFFF0000u));
  }
};

// tanh for scores that are capped: below 0.6 an odd polynomial (least squares at Chebyshev's points; to 2^-26 of the value), else by an exponential (to 2^-22).
__device__ __forceinline__ float tanh_near(float y)
{
  const float z = y * y;
  float p       = fmaf(z, -0.006276390049606562f, 0.021116215735673904f);
  p             = fmaf(z, p, -0.053875137120485306f);
  p             = fmaf(z, p, 0.13332924246788025f);
  p             = fmaf(z, p, -0.3333333134651184f);
  return fmaf(y * z, p, y);
}
__device__ __forceinline__ float tanh_any(float y)
{
  const float e = power_of_2(2.8853900817779268f * fabsf(y));  // 2 log2(e)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
  const float t = copysignf(fmaf(-2.0f, r, 1.0f), y);
  return fabsf(y) < 0.6f ? tanh_near(y) : t;
}

}  // namespace cuvs_b200::kv
