// Routing to experts: the top_k of E experts for every token, and their weights.
//   p = softmax(logits) or 1 / (1 + exp(-logits));  v = p + bias;  the top_k largest v of the experts in the topk_group best
//   groups (a group's value: the sum of its two largest v), ties to the lowest index;  w = p[ids] (/ sum of them) * scaling.
// Scores, biased scores and group sums are binary64: which of two near values is larger decides an expert, and two evaluations
// of the same scores in 32 bits would choose differently about once in ten thousand tokens (256 experts).
//
// One wavefront per token; lane l holds experts l * EPL .. + EPL - 1 (neighbouring ones, so that a lane's logits are one load and
// the first lane with the largest value holds the lowest index).  The scores also lie in LDS, for the group sums and for the
// weights at the end.
//   8192 tokens, 256 experts, sigmoid, 8 groups: 14.6 us where reading the logits takes 1.8.  All wavefronts are on the machine at once; what bounds
// them is the issue of 870 vector instructions a token: about a quarter each are the scores (binary64 exponentials and reciprocals), the groups and the eight
// choices.  The choices with binary64 maxima over all lanes, the groups scanned by one lane each: 19.5 us.
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
  int lanes_shift;  // 2^lanes_shift lanes for a group
  int group_size;
  uint32_t per_size;  // ceil(2^32 / group_size), for the group of an expert; 0 for groups of one
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

// The largest of the 64 lanes' values.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define TLQ_DPP_MAX(ctrl)                                                                             \
  {                                                                                                   \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);        \
    v = v > o ? v : o;                                                                                \
  }
  TLQ_DPP_MAX(0xb1)
  TLQ_DPP_MAX(0x4e)
  TLQ_DPP_MAX(0x141)
  TLQ_DPP_MAX(0x140)
#undef TLQ_DPP_MAX
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16), c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}
// Whole numbers in the order of the values (no NaN, no -0); 0 is free for an expert that is not to be had.
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t b = bitcast<uint64_t>(v);
  return b ^ ((uint64_t)((int64_t)b >> 63) | ((uint64_t)1 << 63));
}

// 1 / x to about an ulp, x from 1 to 1e300: two of Newton's steps
__device__ __forceinline__ double reciprocal(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
}

template <typename T, int EPL>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(const RouteArgs a) {
  __shared__ double scores[kRouteWaves][64 * EPL];
  __shared__ double values[kRouteWaves][64 * EPL];  // biased, for the group sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (m >= a.M) return;  // (a wavefront shares nothing with the others: no barrier below)
  const double inf = __builtin_huge_val();
  const auto larger = [](double x, double y) { return x > y ? x : y; };
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
    for (int i = 0; i < EPL; ++i) p[i] = 1.0 + exp(masked[i] ? 0.0 : -v[i]);  // (all of them, so that they share their constants)
    bool far = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) far = far || p[i] > 1e300;
    if (__builtin_amdgcn_ballot_w64(far)) {  // (the steps below would lose what is left of such a reciprocal)
#pragma unroll
      for (int i = 0; i < EPL; ++i) p[i] = 1.0 / p[i];
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) p[i] = reciprocal(p[i]);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] = masked[i] ? 0.0 : p[i];
  } else {
    double top = v[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) top = larger(top, v[i]);
    top = wave_all(top, larger);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const bool is_top = v[i] == top;  // (also where both are +infinity)
      p[i] = exp(is_top ? 0.0 : v[i] - top);
      p[i] = masked[i] ? 0.0 : p[i];
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
    // 64 / n_group lanes (a power of two) scan a group in turn, then join their two largest
    const int size = a.group_size, shift = a.lanes_shift, mine = lane >> shift, per = 1 << shift;
    double first = -inf, second = -inf;
    if (mine < a.n_group) {
      for (int i = lane & (per - 1); i < size; i += per) {
        const double y = my_values[mine * size + i];
        second = y > first ? first : y > second ? y : second;
        first = y > first ? y : first;
      }
    }
    for (int o = 1; o < per; o <<= 1) {
      const double f = __shfl_xor(first, o), t = __shfl_xor(second, o);
      const double less = f > first ? first : f, more = t > second ? t : second;
      first = f > first ? f : first;
      second = less > more ? less : more;
    }
    // a group with one expert to be had counts with that one
    const double of_group = second > -inf ? first + second : first;
    int rank = 0;
    const uint64_t bits = bitcast<uint64_t>(of_group);
    for (int g = 0; g < a.n_group; ++g) {
      const double other = from_halves(__builtin_amdgcn_readlane((uint32_t)bits, g << shift), __builtin_amdgcn_readlane((uint32_t)(bits >> 32), g << shift));
      rank += (other > of_group || (other == of_group && g < mine)) ? 1 : 0;
    }
    const uint64_t kept = __builtin_amdgcn_ballot_w64(mine < a.n_group && rank < a.topk_group);  // group g: bit g << shift
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      if (e < a.E && !((kept >> ((a.per_size ? __umulhi((uint32_t)e, a.per_size) : (uint32_t)e) << shift)) & 1)) v[i] = -inf;
    }
  }

  // The largest by the upper halves of the keys, which nearly always one lane alone has; otherwise by the lower halves among those that do.
  uint64_t key[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = v[i] > -inf ? key_of(v[i]) : 0;
  int id = -1;  // lane j: the j-th expert
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t mine = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < EPL; ++i)
      if (key[i] > mine) mine = key[i], at = i;
    const uint32_t upper = (uint32_t)(mine >> 32), best = wave_max(upper);
    if (best == 0) break;  // nothing left: the remaining slots stay empty
    uint64_t have = __builtin_amdgcn_ballot_w64(upper == best);
    if (have & (have - 1)) {
      const uint32_t lower = upper == best ? (uint32_t)mine : 0, best_lower = wave_max(lower);
      have = __builtin_amdgcn_ballot_w64(upper == best && lower == best_lower);
    }
    const int winner = __builtin_ctzll(have);
    const int e = winner * EPL + __builtin_amdgcn_readlane(at, winner);
    if (lane == j) id = e;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane == winner && i == at) key[i] = 0;
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

// (a launch has fewer than 2^32 threads: 2^26 tokens less a work-group's)
constexpr int64_t kRouteTokens = (((int64_t)1 << 24) - 1) * kRouteWaves;

template <typename T>
int run_route(const RouteArgs& all, hipStream_t st) {
  for (int64_t m = 0; m < all.M; m += kRouteTokens) {
    RouteArgs a = all;
    a.logits = (const T*)all.logits + m * all.E;
    a.weights += m * all.top_k, a.ids += m * all.top_k;
    a.M = all.M - m < kRouteTokens ? all.M - m : kRouteTokens;
    const dim3 grid((unsigned)ceil_div(a.M, (int64_t)kRouteWaves));
#define TLQ_ROUTE(EPL) moe_route_kernel<T, EPL><<<grid, 64 * kRouteWaves, 0, st>>>(a)
    if (a.E <= 64) TLQ_ROUTE(1);
    else if (a.E <= 128) TLQ_ROUTE(2);
    else if (a.E <= 256) TLQ_ROUTE(4);
    else if (a.E <= 512) TLQ_ROUTE(8);
    else TLQ_ROUTE(16);
#undef TLQ_ROUTE
    if (!check_launch("tlq_moe_route", "moe_route_kernel")) return 1;
  }
  return 0;
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
  int shift = 6;
  while ((n_group << shift) > 64) --shift;
  const RouteArgs a{logits, (const float*)bias, (float*)weights, (int32_t*)ids, M, (int)E, (int)top_k, (int)n_group, (int)topk_group,
                    scoring == TLQ_MOE_SIGMOID, renormalize != 0, scaling, shift,
                    (int)(E / n_group), E == n_group ? 0u : (uint32_t)ceil_div((int64_t)1 << 32, E / n_group)};
  hipStream_t st = (hipStream_t)stream;
  if (in_dtype == TLQ_F16) return run_route<half_t>(a, st);
  if (in_dtype == TLQ_BF16) return run_route<bf16_t>(a, st);
  return run_route<float>(a, st);
}
