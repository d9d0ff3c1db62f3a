// What the kernels that work on whole rows of activations share (act_quant.hip, norm_act.hip): eight values a load, sums and maxima
// over a wavefront, codes of 8 bits.
#pragma once
#include <type_traits>

#include "tlq_common.h"

namespace tlq {

template <>
__device__ __forceinline__ float to_float<float>(float v) {
  return v;
}

// Eight consecutive values, kept as loaded (16 or 32 bytes) and widened to float on use.  The input is read once:
// non-temporal loads (M = 16384, N = 4096: 38.2 instead of 40.0 us; with the resident grid 36.1 us) -- but for load_shared, whose
// values other work-groups read too.  The output is
// stored normally: non-temporal stores save another microsecond here and cost the W8A8 GEMM that reads the output next
// 4 - 14 us (16384 x 4096 x 4096: quantiser + GEMM 291 against 279 us).
template <typename T>
struct Raw8;
template <>
struct Raw8<half_t> {
  half8_t v;
  __device__ __forceinline__ void load(const half_t* p) { v = __builtin_nontemporal_load((const half8_t*)p); }
  __device__ __forceinline__ void load_shared(const half_t* p) { v = *(const half8_t*)p; }
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
};
template <>
struct Raw8<bf16_t> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const bf16_t* p) {
    const uint4_t q = __builtin_nontemporal_load((const uint4_t*)p);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  }
  __device__ __forceinline__ void load_shared(const bf16_t* p) {
    const uint4_t q = *(const uint4_t*)p;
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  }
  __device__ __forceinline__ float get(int i) const {
    return bitcast<float>((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
  }
};
template <>
struct Raw8<float> {
  float4_t a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __builtin_nontemporal_load((const float4_t*)p);
    b = __builtin_nontemporal_load((const float4_t*)(p + 4));
  }
  __device__ __forceinline__ void load_shared(const float* p) { a = *(const float4_t*)p, b = *(const float4_t*)(p + 4); }
  __device__ __forceinline__ float get(int i) const { return i < 4 ? a[i] : b[i - 4]; }
};

__device__ __forceinline__ float wave_max(float v) {
  // a row of 16 lanes inside the vector unit (lanes swapped in pairs, in fours, halves of a row and rows mirrored), then rows and halves
  // of the wavefront swapped: no trip through LDS
  auto dpp = [&](auto ctrl) { v = fmaxf(v, bitcast<float>(__builtin_amdgcn_update_dpp(0, bitcast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false))); };
  dpp(std::integral_constant<int, 0xb1>{}), dpp(std::integral_constant<int, 0x4e>{}), dpp(std::integral_constant<int, 0x141>{}), dpp(std::integral_constant<int, 0x140>{});
  const auto rows = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
  v = fmaxf(bitcast<float>((uint32_t)rows[0]), bitcast<float>((uint32_t)rows[1]));
  const auto halves = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
  return fmaxf(bitcast<float>((uint32_t)halves[0]), bitcast<float>((uint32_t)halves[1]));
}

__device__ __forceinline__ float row_scale(float amax, int round_scale) {
  amax = fmaxf(amax, 1e-4f);
  const float s = amax / 127.0f;
  if (!round_scale) return s;
  // 2^ceil(log2(s)) from the bits of s: exponent, plus one when any mantissa bit is set
  const uint32_t bits = bitcast<uint32_t>(s);
  const int e = (int)((bits >> 23) & 0xff) - 127 + ((bits & 0x7fffffu) ? 1 : 0);
  return bitcast<float>((uint32_t)(e + 127) << 23);
}

// x / scale, correctly rounded wherever the quotient matters, from the row's reciprocal
// rcp = fl(1 / scale): q0 = x * rcp is within an ulp, the remainder x - q0 * scale is exact in one
// fma, and one more fma lands on the correctly rounded quotient.  (Only when the remainder
// underflows, |x| < 2^-100 or so, can the last bit differ; such quotients round to 0 either way.)
__device__ __forceinline__ uint32_t quant1(float x, float scale, float rcp) {
  const float q0 = x * rcp;
  const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, scale, x), rcp, q0);
  // bounded (NaN becomes the lower bound), then to the nearest even whole number by the addition, which leaves its two's complement in
  // the low byte
  return bitcast<uint32_t>(__builtin_amdgcn_fmed3f(q1, -127.0f, 127.0f) + 12582912.0f);
}

template <typename R>
__device__ __forceinline__ uint2_t quant8(const R& r, float scale, float rcp) {
  uint2_t o;
  auto four = [&](int i) {
    const uint32_t lo = __builtin_amdgcn_perm(quant1(r.get(i + 1), scale, rcp), quant1(r.get(i), scale, rcp), 0x0c0c0400u);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(quant1(r.get(i + 3), scale, rcp), quant1(r.get(i + 2), scale, rcp), 0x0c0c0400u), lo, 0x05040100u);
  };
  o.x = four(0), o.y = four(4);
  return o;
}

}  // namespace tlq
