// What the kernels of the experts' products share (moe_w4a16.hip, moe_w4a16_panel.hip).
#pragma once
#include "expand8.h"
#include "gemm_core.h"
#include "silu.h"

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
