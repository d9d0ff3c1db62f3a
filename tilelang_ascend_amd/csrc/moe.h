// What the kernels of the experts' products share (moe_w4a16.hip, moe_w4a16_panel.hip).
#pragma once
#include "expand8.h"
#include "gemm_core.h"

namespace tlq {

// A tile of pairs: `pairs` of them, those of `expert` from entry `first` of the sorted pairs on; expert E: pairs without an expert.
struct PlanTile {
  int32_t expert, first, pairs, unused;
};
// What a call works out of its ids: the pairs by expert, tiles of few pairs, tiles of 256 pairs, and how many of either there are.
struct Plan {
  const int32_t* order;
  const PlanTile *small, *large;
  const int32_t* totals;  // [0] small, [1] large
};
constexpr int kLargeRows = 256;
constexpr int64_t kMostGroups = ((int64_t)1 << 24) - 1;  // work-groups of 256 threads of a launch, which has fewer than 2^32 threads

struct ExpertArgs {
  const void* X;         // activations: [M, K] (gate / up) or [pairs, K] (down)
  const uint8_t* Wp;     // [E, rows of an expert, K / 2]
  const void* scales;    // [E, rows of an expert, K / group] or null
  const void* zeros;     // the same, or null
  const float* weights;  // down: [pairs]
  void* out;             // gate / up: h [pairs, N]; down: fp32 [pairs, N]
  int E, top_k, N, K, group;
  float zero_scalar;
};

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

// Gate / up (up = true) or down product of the tiles of 256 pairs (moe_w4a16_panel.hip).
bool moe_panel_takes(const ExpertArgs& a, int64_t pairs, bool up);
int64_t moe_panel_groups(int64_t N, bool up);  // work-groups of a tile
int moe_panel(const char* what, const ExpertArgs& a, const Plan& plan, int64_t most_tiles, int dtype, bool up, hipStream_t st);

// Four neighbouring sums of one pair: gate / up: outputs n .. n + 3 from the gates in q = 0, 1 and their ups 32 lanes on; down: the weighted row.
template <typename T, bool UP, typename Args>
__device__ __forceinline__ void moe_store(const Args& a, const float4_t& sum, bool live, int pair, float weight, int n, int q, int chunk) {
  if constexpr (UP) {
    float4_t up;
#pragma unroll
    for (int i = 0; i < 4; ++i) up[i] = __shfl_xor(sum[i], 32);
    if (q < 2 && live) {
      const float4_t y = silu_times(sum, up);
      T o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = from_float<T>(y[i]);
      *(uint2_t*)((T*)a.out + (int64_t)pair * a.N + n) = bitcast<uint2_t>(o);
    }
  } else if (live) {
    *(float4_t*)((float*)a.out + ((int64_t)chunk * a.pairs + pair) * a.N + n) = sum * weight;
  }
}

}  // namespace tlq
