// The gated activation of an MLP (moe.h: the experts' products, norm_act.hip: behind a dense product).
#pragma once
#include "tlq_common.h"

namespace tlq {

// silu(x) * u, silu(x) = x / (1 + exp(-x)) (the reciprocal to an ulp).  From x = -87 on the reciprocal is less than fp32 holds, and then exp(-x) more,
// where the product is still a normal number (bfloat16 has fp32's range): x u e^2 / (1 + e^2) there, e = exp(x / 2), one e at the end.  A value goes by
// its own x; the branch only saves the second way where no lane needs it (gate / up of 65536 pairs of 64 experts of 1024 x 2048: 558 us, 566 with
// e for all x, 559 without either).
__device__ __forceinline__ float4_t silu_times(const float4_t& x, const float4_t& u) {
  float4_t y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-x[i])) * u[i];
  const float a = x[0] < x[1] ? x[0] : x[1], b = x[2] < x[3] ? x[2] : x[3];  // (NaN where the second of two is one)
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(a >= -80.0f) || !(b >= -80.0f)) != 0, 0)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = __expf(0.5f * x[i]), far = e * __builtin_amdgcn_rcpf(1.0f + e * e) * x[i] * u[i] * e;
      y[i] = x[i] < -80.0f ? far : y[i];
    }
  }
  return y;
}

}  // namespace tlq
