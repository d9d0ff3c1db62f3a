// Routing to experts: the top_k of E experts for every token, and their weights.
//   p = softmax(logits) or 1 / (1 + exp(-logits));  v = p + bias;  the top_k largest v of the experts in the topk_group best
//   groups (a group's value: the sum of its two largest v), ties to the lowest index;  w = p[ids] (/ sum of them) * scaling.
// Scores, biased scores and group sums are binary64: which of two near values is larger decides an expert, and two evaluations
// of the same scores in 32 bits would choose differently about once in ten thousand tokens (256 experts).
//
// One wavefront per token; lane l holds experts l * EPL .. + EPL - 1 (neighbouring ones, so that a lane's logits are one load and
// the first lane with the largest value holds the lowest index).  The scores also lie in LDS, for the group sums and for the
// weights at the end.
#include "tlq_common.h"

namespace tlq {

template <>
__device__ __forceinline__ float to_float<float>(float v) {
  return v;
}

namespace {

constexpr int kRouteWaves = 4;

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  int64_t M;
  int E, top_k, n_group, topk_group;
  int sigmoid, renormalize;
  float scaling;
};

__device__ __forceinline__ double from_halves(uint32_t lo, uint32_t hi) { return bitcast<double>(((uint64_t)hi << 32) | lo); }

// op over the 64 lanes, the same result in every lane: lanes swapped in pairs, in fours, halves of a row and rows mirrored, then rows
// and halves of the wavefront swapped.  The order of the operands is the same in every call: sums do not depend on timing.
template <typename Op>
__device__ __forceinline__ double wave_all(double v, Op op) {
#define TLQ_DPP64(ctrl)                                                                                    \
  {                                                                                                        \
    const uint64_t b = bitcast<uint64_t>(v);                                                               \
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl, 0xf, 0xf, false);           \
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), ctrl, 0xf, 0xf, false);   \
    v = op(v, from_halves(lo, hi));                                                                        \
  }
  TLQ_DPP64(0xb1)
  TLQ_DPP64(0x4e)
  TLQ_DPP64(0x141)
  TLQ_DPP64(0x140)
#undef TLQ_DPP64
  {
    const uint64_t b = bitcast<uint64_t>(v);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    v = op(from_halves(lo[0], hi[0]), from_halves(lo[1], hi[1]));
  }
  {
    const uint64_t b = bitcast<uint64_t>(v);
    const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    v = op(from_halves(lo[0], hi[0]), from_halves(lo[1], hi[1]));
  }
  return v;
}

template <typename T, int EPL>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(const RouteArgs a) {
  __shared__ double scores[kRouteWaves][64 * EPL];
  __shared__ double values[kRouteWaves][64 * EPL];  // biased, for the group sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (m >= a.M) return;  // (a wavefront shares nothing with the others: no barrier below)
  const double inf = __builtin_huge_val();
  const auto larger = [](double x, double y) { return __builtin_fmax(x, y); };
  const auto plus = [](double x, double y) { return x + y; };
  double* const my_scores = scores[wave];
  double* const my_values = values[wave];

  const T* const x = (const T*)a.logits + m * a.E;
  double v[EPL], p[EPL];
  bool masked[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    const float f = e < a.E ? to_float(x[e]) : -__builtin_inff();
    masked[i] = !(f > -__builtin_inff());  // -infinity and NaN: an expert that is not to be had
    v[i] = masked[i] ? -inf : (double)f;
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] = masked[i] ? 0.0 : 1.0 / (1.0 + exp(-v[i]));
  } else {
    double top = v[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) top = larger(top, v[i]);
    top = wave_all(top, larger);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      p[i] = masked[i] ? 0.0 : v[i] == top ? 1.0 : exp(v[i] - top);  // (equal: also where both are +infinity)
      sum += p[i];
    }
    sum = wave_all(sum, plus);
    const double scale = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] *= scale;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    my_scores[e] = p[i];
    double biased = p[i];
    if (a.bias && e < a.E) biased += (double)a.bias[e];
    v[i] = masked[i] || !(biased > -inf) ? -inf : biased;  // (a bias of -infinity or NaN masks as well)
  }

  if (a.n_group > 1) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) my_values[lane * EPL + i] = v[i];
    __builtin_amdgcn_wave_barrier();
    const int size = a.E / a.n_group;
    double first = -inf, second = -inf;
    if (lane < a.n_group) {
      int at = lane % size;  // (every lane starts elsewhere: the groups are whole multiples of the banks apart)
      for (int i = 0; i < size; ++i) {
        const double y = my_values[lane * size + at];
        at = at + 1 == size ? 0 : at + 1;
        second = larger(second, __builtin_fmin(first, y));
        first = larger(first, y);
      }
    }
    // a group with one expert to be had counts with that one
    const double of_group = second > -inf ? first + second : first;
    int rank = 0;
    const uint64_t bits = bitcast<uint64_t>(of_group);
    for (int g = 0; g < a.n_group; ++g) {
      const double other = from_halves(__builtin_amdgcn_readlane((uint32_t)bits, g), __builtin_amdgcn_readlane((uint32_t)(bits >> 32), g));
      rank += (other > of_group || (other == of_group && g < lane)) ? 1 : 0;
    }
    const uint64_t kept = __builtin_amdgcn_ballot_w64(lane < a.n_group && rank < a.topk_group);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      if (e < a.E && !((kept >> (e / size)) & 1)) v[i] = -inf;
    }
  }

  int id = -1;  // lane j: the j-th expert
  for (int j = 0; j < a.top_k; ++j) {
    double mine = v[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < EPL; ++i)
      if (v[i] > mine) mine = v[i], at = i;
    const double best = wave_all(mine, larger);
    if (!(best > -inf)) break;  // nothing left: the remaining slots stay empty
    const int winner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine == best));
    const int e = winner * EPL + __builtin_amdgcn_readlane(at, winner);
    if (lane == j) id = e;
    if (lane == winner) {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i == at) v[i] = -inf;
    }
  }
  __builtin_amdgcn_wave_barrier();
  double w = id >= 0 ? my_scores[id] : 0.0;
  if (a.renormalize) {
    const double sum = wave_all(w, plus);
    w = sum > 0.0 ? w / sum : 0.0;
  }
  if (lane < a.top_k) {
    a.weights[m * a.top_k + lane] = (float)(w * (double)a.scaling);
    a.ids[m * a.top_k + lane] = id;
  }
}

template <typename T>
int run_route(const RouteArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.M, (int64_t)kRouteWaves));
#define TLQ_ROUTE(EPL) moe_route_kernel<T, EPL><<<grid, 64 * kRouteWaves, 0, st>>>(a)
  if (a.E <= 64) TLQ_ROUTE(1);
  else if (a.E <= 128) TLQ_ROUTE(2);
  else if (a.E <= 256) TLQ_ROUTE(4);
  else if (a.E <= 512) TLQ_ROUTE(8);
  else TLQ_ROUTE(16);
#undef TLQ_ROUTE
  return check_launch("tlq_moe_route", "moe_route_kernel") ? 0 : 1;
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int tlq_moe_route(const void* logits, const void* bias, void* weights, void* ids, int64_t M, int64_t E, int64_t top_k,
                             int64_t n_group, int64_t topk_group, int scoring, int renormalize, float scaling, int in_dtype,
                             void* stream) {
  TLQ_REQUIRE(M >= 0 && M < ((int64_t)1 << 32) && E >= 1 && E <= 1024, "tlq_moe_route: bad shape M=%lld E=%lld (at most 1024 experts)",
              (long long)M, (long long)E);
  TLQ_REQUIRE(n_group >= 1 && n_group <= 64 && E % n_group == 0, "tlq_moe_route: n_group=%lld must divide E=%lld and be at most 64",
              (long long)n_group, (long long)E);
  TLQ_REQUIRE(topk_group >= 1 && topk_group <= n_group, "tlq_moe_route: topk_group=%lld must be 1 .. n_group=%lld", (long long)topk_group,
              (long long)n_group);
  TLQ_REQUIRE(top_k >= 1 && top_k <= 64 && top_k <= E / n_group * topk_group,
              "tlq_moe_route: top_k=%lld must be at most 64 and at most the %lld experts of the chosen groups", (long long)top_k,
              (long long)(E / n_group * topk_group));
  TLQ_REQUIRE(scoring == TLQ_MOE_SOFTMAX || scoring == TLQ_MOE_SIGMOID, "tlq_moe_route: unknown scoring %d", scoring);
  TLQ_REQUIRE(in_dtype == TLQ_F16 || in_dtype == TLQ_BF16 || in_dtype == TLQ_F32,
              "tlq_moe_route: in_dtype must be float16, bfloat16 or float32 (got %d)", in_dtype);
  if (M == 0) return 0;
  TLQ_REQUIRE(logits && weights && ids, "tlq_moe_route: null pointer");
  TLQ_REQUIRE((((uintptr_t)weights | (uintptr_t)ids | (uintptr_t)bias) & 3) == 0 && ((uintptr_t)logits & (in_dtype == TLQ_F32 ? 3 : 1)) == 0,
              "tlq_moe_route: misaligned pointer");
  const RouteArgs a{logits, (const float*)bias, (float*)weights, (int32_t*)ids, M, (int)E, (int)top_k, (int)n_group, (int)topk_group,
                    scoring == TLQ_MOE_SIGMOID, renormalize != 0, scaling};
  hipStream_t st = (hipStream_t)stream;
  if (in_dtype == TLQ_F16) return run_route<half_t>(a, st);
  if (in_dtype == TLQ_BF16) return run_route<bf16_t>(a, st);
  return run_route<float>(a, st);
}
