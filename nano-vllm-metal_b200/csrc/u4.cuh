// u4.cuh -- the 4-bit cache's row format, shared by the kernels that write, read and attend to it.
//
// A row (one token of one kv head, D = 64 or 128 elements) is D/2 bytes of codes and D/64 pairs of
// (scale s, offset z) of a 16-bit type T, one pair for each group of 64 elements:
//   byte j = code of element 2j | code of element 2j + 1 << 4,      value = s * code + z.
// z is the group's least value (rounded toward -inf where T is narrower than the input), s a
// fifteenth of the span above z rounded toward +inf: every element then lies on [z, z + 15 s], so
// none is off by more than half a step (nearest rounding of s would clip the top of one group in
// two, by up to 15 half ulps of s).  code = clip(rint(fl((x - z) / s)), 0, 15), 0 where s = 0.  A
// group that holds a NaN or an infinity, or whose span is none of T's numbers, reads back as NaN.
#pragma once

#include "nvm_common.cuh"

namespace nvm {

constexpr int kU4Group = 64;

// x / 15 rounded to nearest: a product with the rounded inverse is within an ulp of the quotient, and one
// correction by the exact remainder then rounds as the division does (Markstein), at a third of its
// instructions; quotients near the subnormals divide.  NaN and infinities give NaN.
__device__ __forceinline__ float over15(float x) {
  if (x < 0x1p-100f) return __fdiv_rn(x, 15.0f);
  const float q = __fmul_rn(x, 1.0f / 15.0f);
  return __fmaf_rn(__fmaf_rn(-15.0f, q, x), 1.0f / 15.0f, q);
}

// The pair (s, z) of a group from its extremes, in fp32 with the values that T holds; s = z = NaN
// for a group that cannot be held.
template <typename T>
__device__ __forceinline__ float2 u4_scale(float lo, float hi);
template <>
__device__ __forceinline__ float2 u4_scale<__nv_bfloat16>(float lo, float hi) {
  const float z = __bfloat162float(__float2bfloat16_rd(lo));
  const float s = __bfloat162float(__float2bfloat16_ru(over15(__fsub_rn(hi, z))));
  const bool ok = s < INFINITY && z > -INFINITY;  // false for NaN too
  return ok ? make_float2(s, z) : make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
}
template <>
__device__ __forceinline__ float2 u4_scale<__half>(float lo, float hi) {
  const float z = __half2float(__float2half_rd(lo));
  const float s = __half2float(__float2half_ru(over15(__fsub_rn(hi, z))));
  const bool ok = s < INFINITY && z > -INFINITY;
  return ok ? make_float2(s, z) : make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
}

// 1 / s for u4_code_fast, within an ulp (0 where the group has no steps: every code is then 0; infinite
// for the least subnormals, whose codes are then divided).
__device__ __forceinline__ float u4_inverse(float s) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
  return s > 0.0f ? r : 0.0f;
}

// code of x.  t = fl(d * r) with r within 2^-23 of 1 / s is within 15 (2^-23 + 2^-24 + 2^-24) < 2^-18 of
// fl(d / s) for quotients up to 15 (1 + 2^-23), so where t is at least 2^-14 from every half-integer both round to the same integer; `amb` marks
// the others (and NaN) for u4_code_div.
__device__ __forceinline__ int u4_code_fast(float x, float z, float r, bool& amb) {
  const float t = __fmul_rn(__fsub_rn(x, z), r);
  const float f = __fadd_rn(t, 12582912.0f);
  amb = !(fabsf(__fsub_rn(t, __fsub_rn(f, 12582912.0f))) < 0.5f - 0x1p-14f);
  return min(max(__float_as_int(f) - 0x4B400000, 0), 15);
}
__device__ __forceinline__ int u4_code_div(float x, float z, float s) {
  const float y = rintf(__fdiv_rn(__fsub_rn(x, z), s));
  return (int)fminf(fmaxf(y, 0.0f), 15.0f);  // NaN (0 / 0, a group that cannot be held) gives 0
}

// Two 16-bit numbers of the scale type as they lie in memory (s low, z high), in fp32.
template <typename T>
__device__ __forceinline__ float2 u4_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 u4_pair<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 u4_pair<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// (s, z) packed as they lie in memory; both are values of T.
template <typename T>
__device__ __forceinline__ uint32_t u4_pack_pair(float2 sz) {
  return pack2<T>(sz.x, sz.y);
}

// Division of numbers below 2^31 by one of 1 .. 2^31 that a launch knows.  With 2^(k - 1) < d <= 2^k and
// mul = floor(2^(31 + k) / d) + 1 the error mul * d - 2^(31 + k) is at most 2^k, so n * mul >> 31 + k is exact.
struct FastDiv {
  uint32_t mul, shift;
  FastDiv() = default;
  explicit FastDiv(int64_t d) {
    int k = 0;
    while ((int64_t(1) << k) < d) ++k;
    mul = (uint32_t)((uint64_t(1) << (31 + k)) / (uint64_t)d + 1);
    shift = (uint32_t)(31 + k);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((uint64_t)n * mul >> shift); }
};

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

}  // namespace nvm
