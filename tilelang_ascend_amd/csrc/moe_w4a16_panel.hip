// The experts' products on tiles of 256 pairs: the step loop of the 256-row W4A16 kernel (panel256.h) with the rows of a tile gathered through
// the plan's sorted pairs, an expert's matrix as the weights, and epilogues of its own.
//   gate / up: a work-group has 128 outputs; wavefront w the 32 from 32 w on, its weight tiles 0, 1 being their gate rows and 2, 3 their
// up rows, so that gate and up of an output meet in one lane.  down: 256 outputs, 64 a wavefront; weighted fp32 rows.
// Work-groups in the order of the tiles, those of one tile next to each other, and every XCD a contiguous range of them: 32 at a time, that share
// a few tiles' activation rows and one expert's weights in its L2.
//   bf16, one zero point, 65536 pairs of 64 experts of 1024 x 2048 (gate / up): 519 - 549 us by the tracer on two boxes, 1.0 - 1.06 PFLOP/s of the pairs' own
// products; the rate of the step loop alone is that of the dense product, 1.3 - 1.35 (power), the difference the rows that fill up an expert's last tile and
// the last round of work-groups.
#include "moe.h"
#include "panel256.h"

namespace tlq {
namespace {

struct PanelArgs {
  const void* X;
  const uint8_t* Wp;
  const void* scales;
  const void* zeros;
  const float* weights;
  void* out;
  const int32_t* order;
  const PlanTile* tiles;
  const int32_t* total;
  int top_k, N, K, gshift, n_groups;
  float zero_scalar;
};

template <typename T, bool UP, int ZM>
__global__ __launch_bounds__(256, 1) void moe_panel_kernel(const PanelArgs a) {
  typedef Panel2Cfg Cfg;
  constexpr int TM = Cfg::TM, TN = Cfg::TN, LA = Cfg::LA;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const int live = *a.total * a.n_groups;
  if ((int)blockIdx.x >= live) return;
  const int no = addr::xcd_order(blockIdx.x, live);
  const int tile_no = (int)((uint32_t)no / (uint32_t)a.n_groups), group_no = no - tile_no * a.n_groups;
  const PlanTile pt = a.tiles[tile_no];
  const int e = __builtin_amdgcn_readfirstlane(pt.expert), rows = __builtin_amdgcn_readfirstlane(pt.pairs);
  if (rows == 0) return;
  const int32_t* const mine = a.order + __builtin_amdgcn_readfirstlane(pt.first);
  const int groups = a.K >> a.gshift;
  const int64_t row0 = (int64_t)e * (UP ? 2 : 1) * a.N;  // of the expert's matrix

  // (the host has checked that what the offsets reach is below 4 GiB)
  uint32_t voff_a[LA], voff_w[TN], voff_sc[TN];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = 4 * (j * 4 + wave) + (lane >> 4), pair = mine[r < rows ? r : rows - 1];
    voff_a[j] = (uint32_t)(UP ? pair / a.top_k : pair) * (uint32_t)(a.K * 2) + addr::panel_a_chunk(lane, wave);
  }
  const int n0 = group_no * (UP ? Cfg::BN / 2 : Cfg::BN);
  // weight rows of tile tn of a wavefront begin at n_of(tn); past the matrix its last ones, whose outputs are not stored
  auto n_of = [&](int tn) { return UP ? n0 + wave * 32 + (tn & 1) * 16 : n0 + wave * 64 + tn * 16; };
#pragma unroll
  for (int tn = 0; tn < TN; ++tn) {
    int n = n_of(tn);
    n = n + 16 <= a.N ? n : a.N - 16;
    if (UP && tn >= 2) n += a.N;
    voff_w[tn] = (uint32_t)n * (uint32_t)(a.K >> 1) + addr::panel_w_lane(lane, a.K);
    voff_sc[tn] = (uint32_t)n * (uint32_t)(groups * 2) + addr::panel2_sc_lane(lane, groups, a.gshift);
  }
  const T* const scales = a.scales ? (const T*)a.scales + row0 * groups : nullptr;
  const T* const zeros = ZM == 0 ? (const T*)a.zeros + row0 * groups : nullptr;
  typename Panel2Mma<T>::acc_t acc[TN][TM];
  panel256_steps<T, 0, ZM>(smem, (const T*)a.X, a.Wp + row0 * (a.K >> 1), scales, zeros, voff_a, voff_w, voff_sc, 0, a.K >> 7, a.gshift, a.zero_scalar, acc);

  // lane (r16, q) holds row 16 tm + r16, weight rows n_of(tn) + 4 q .. + 3
#pragma unroll
  for (int tm = 0; tm < TM; ++tm) {
    const int r = tm * 16 + r16;
    const bool live_row = r < rows;
    const int pair = mine[live_row ? r : rows - 1];
    if constexpr (UP) {
      T* const h = (T*)a.out + (int64_t)pair * a.N;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float4_t g = acc[t][tm], u = acc[t + 2][tm];
        asm volatile("" : "+v"(g), "+v"(u));  // (moved out of the accumulation registers here, not all of them ahead)
        const int n = n_of(t) + q * 4;
        const float4_t y = silu_times(g, u);
        T o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = from_float<T>(y[i]);
        if (live_row && n < a.N) *(uint2_t*)(h + n) = bitcast<uint2_t>(o);
      }
    } else {
      float* const y = (float*)a.out + (int64_t)pair * a.N;
      const float weight = a.weights[pair];
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) {
        float4_t v = acc[tn][tm];
        asm volatile("" : "+v"(v));
        const int n = n_of(tn) + q * 4;
        if (live_row && n < a.N) *(float4_t*)(y + n) = v * weight;
      }
    }
  }
}

template <typename T, bool UP, int ZM>
int launch_panel(const char* what, const PanelArgs& a, int64_t grid, hipStream_t st) {
  auto kern = moe_panel_kernel<T, UP, ZM>;
  static bool attr_set = false;
  if (!attr_set) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, Panel2Cfg::LDS);
    TLQ_REQUIRE(e == hipSuccess, "%s: cannot reserve %d bytes of LDS: %s", what, (int)Panel2Cfg::LDS, hipGetErrorString(e));
    attr_set = true;
  }
  kern<<<(unsigned)grid, 256, Panel2Cfg::LDS, st>>>(a);
  return check_launch(what, "moe_panel_kernel") ? 0 : 1;
}

}  // namespace

// Whole steps of 128 values, groups of a power of two, and 32-bit offsets inside an expert's matrix and the activations.
bool moe_panel_takes(const ExpertArgs& a, int64_t pairs, bool up) {
  const int64_t reach = (int64_t)1 << 32, x_rows = up ? pairs / a.top_k : pairs;
  return a.K % 128 == 0 && (a.group & (a.group - 1)) == 0 && x_rows * a.K * 2 < reach && (up ? 2 : 1) * (int64_t)a.N * (a.K / 2) < reach;
}

int64_t moe_panel_groups(int64_t N, bool up) { return ceil_div(N, (int64_t)(up ? Panel2Cfg::BN / 2 : Panel2Cfg::BN)); }

int moe_panel(const char* what, const ExpertArgs& x, const Plan& plan, int64_t most_tiles, int dtype, bool up, hipStream_t st) {
  int gshift = 0;
  while ((1 << gshift) < x.group) ++gshift;
  const int64_t n_groups = moe_panel_groups(x.N, up), grid = most_tiles * n_groups;
  TLQ_REQUIRE(grid <= kMostGroups, "%s: %lld work-groups: call it for fewer tokens at once", what, (long long)grid);
  const PanelArgs a{x.X, x.Wp, x.scales, x.zeros, x.weights, x.out, plan.order, plan.large, plan.totals + 1, x.top_k, x.N, x.K, gshift, (int)n_groups, x.zero_scalar};
  const bool whole = zero_folds(x.zero_scalar);
#define TLQ_PANEL2(T, UP) (x.zeros ? launch_panel<T, UP, 0>(what, a, grid, st) : whole ? launch_panel<T, UP, 1>(what, a, grid, st) : launch_panel<T, UP, 2>(what, a, grid, st))
#define TLQ_PANEL(T) (up ? TLQ_PANEL2(T, true) : TLQ_PANEL2(T, false))
  return dtype == TLQ_F16 ? TLQ_PANEL(half_t) : TLQ_PANEL(bf16_t);
#undef TLQ_PANEL
#undef TLQ_PANEL2
}

}  // namespace tlq
