// Rows of a paged cache of keys and values on the device: 16-byte pieces as floats, places of slots, powers of two.
#pragma once

#include "kv_cache.hpp"
#include "kv_place.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cuvs_b200::kv {

constexpr unsigned kAllLanes = 0xFFFFFFFFu;
constexpr float kLog2E       = 1.4426950408889634f;
constexpr float kLn2         = 0.6931471805599453f;

template <typename T>
constexpr int kPerPiece = 16 / int(sizeof(T));  // elements of a 16-byte piece

template <typename T>
__device__ __forceinline__ void piece_to_floats(const uint4& w, float* f);
template <>
__device__ __forceinline__ void piece_to_floats<float>(const uint4& w, float* f)
{
  f[0] = __uint_as_float(w.x);
  f[1] = __uint_as_float(w.y);
  f[2] = __uint_as_float(w.z);
  f[3] = __uint_as_float(w.w);
}
template <>
__device__ __forceinline__ void piece_to_floats<__half>(const uint4& w, float* f)
{
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
    f[2 * i]       = t.x;
    f[2 * i + 1]   = t.y;
  }
}
template <>
__device__ __forceinline__ void piece_to_floats<__nv_bfloat16>(const uint4& w, float* f)
{
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i]     = __uint_as_float(v[i] << 16);
    f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}

// rounded to the nearest, once
template <typename T>
__device__ __forceinline__ uint4 floats_to_piece(const float* f);
template <>
__device__ __forceinline__ uint4 floats_to_piece<float>(const float* f)
{
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <>
__device__ __forceinline__ uint4 floats_to_piece<__half>(const float* f)
{
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    v[i]            = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ uint4 floats_to_piece<__nv_bfloat16>(const float* f)
{
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    v[i]                   = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x)
{
  return x;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x)
{
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x)
{
  return __float2bfloat16_rn(x);
}

// A 16-byte load that is made or not without a branch, so that several of them are in flight together; 0 where it is not made.
__device__ __forceinline__ uint4 load_piece(const void* from, bool there)
{
  uint4 v;
  asm volatile(
    "{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n mov.u32 %0, 0;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n mov.u32 %3, 0;\n"
    " @p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
    : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
    : "l"(from), "r"(uint32_t(there))
    : "memory");
  return v;
}

// Page and place in it of a slot.
__device__ __forceinline__ void split_slot(const cache_view& c, int64_t slot, uint32_t& page, uint32_t& place)
{
  if (uint64_t(slot) >> 31 == 0) {
    split_place(uint32_t(slot), c.page, page, place);
  } else {
    page  = uint32_t(slot / int64_t(c.page.size));
    place = uint32_t(slot - int64_t(page) * int64_t(c.page.size));
  }
}

// 2^x, to 2^-22 of its value; below 2^-126 it is 0.
__device__ __forceinline__ float power_of_2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(score - top) where nothing is an answer too: top = -inf leaves every weight 0.
__device__ __forceinline__ float finite_top(float top) { return top == -INFINITY ? 0.0f : top; }

}  // namespace cuvs_b200::kv
