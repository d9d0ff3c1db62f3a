// The experts' products of a mixture-of-experts layer on packed 4-bit weights.
//   gate / up:  h[t, j, n] = silu(x[t] . W[e, n]) * (x[t] . W[e, N + n]),  e = ids[t, j]
//   down:       y[t, n] = sum_j w[t, j] * (h[t, j] . W[e, n])
// W = rn_T(rn_T(T(u) - z) * s) as everywhere in this library, fp32 sums.  A pair (t, j) whose id names no expert has h = 0 and
// adds nothing.
//
// Pairs are sorted by expert first (moe_plan_kernel: counts, where each expert's pairs begin, the pairs in order -- a pair keeps
// its place among those of its expert, so nothing depends on timing), then every expert's rows are cut into tiles of activation
// rows, which work-groups find by their number.
#include "expand8.h"
#include "gemm_core.h"

namespace tlq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxExperts = 1024;

// What a call works out of its ids, in the workspace:
//   begin[E + 2]  where the pairs of expert e begin in `order`; entry E: those without an expert, entry E + 1: the number of pairs
//   tiles[E + 2]  the same for tiles of `rows` pairs
//   order[P]      pairs by expert
struct PlanPtrs {
  int32_t *begin, *tiles, *order;
};
__host__ __device__ inline int64_t plan_bytes(int64_t E, int64_t pairs) { return (((E + 2) * 2 + pairs) * 4 + 255) / 256 * 256; }
inline PlanPtrs plan_at(void* ws, int64_t E) {
  int32_t* p = (int32_t*)ws;
  return {p, p + (E + 2), p + 2 * (E + 2)};
}

// One work-group per expert, and one more for the pairs without one: each counts all pairs (LDS histogram; whole numbers, so the
// order of the atomic adds does not matter) and writes down its own.
__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ begin,
                                                               int32_t* __restrict__ tiles, int32_t* __restrict__ order, int pairs,
                                                               int E, int rows) {
  __shared__ int32_t count[kMaxExperts + 1];
  __shared__ int32_t part[kPlanThreads / 64][2];
  __shared__ int32_t of_wave[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = blockIdx.x;
  constexpr int waves = kPlanThreads / 64;
  for (int i = tid; i <= E; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  // every wavefront takes a run of pairs, so that a pair's place is that of its wavefront, its step and its lane
  const int steps = (pairs + kPlanThreads - 1) / kPlanThreads;
  const int first = wave * steps * 64;
  int mine = 0;
  for (int s = 0; s < steps; ++s) {
    const int p = first + s * 64 + lane;
    if (p < pairs) {
      const int id = ids[p];
      const int at = (uint32_t)id < (uint32_t)E ? id : E;
      atomicAdd(&count[at], 1);
      mine += at == e;
    }
  }
  // pairs of this expert in the wavefront's run
  for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
  if (lane == 0) of_wave[wave] = mine;
  __syncthreads();
  // pairs and tiles of the experts before this one
  int before = 0, tiles_before = 0;
  for (int i = tid; i < e; i += kPlanThreads) before += count[i], tiles_before += (count[i] + rows - 1) / rows;
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o), tiles_before += __shfl_xor(tiles_before, o);
  if (lane == 0) part[wave][0] = before, part[wave][1] = tiles_before;
  __syncthreads();
  before = tiles_before = 0;
  int at = 0;
#pragma unroll
  for (int i = 0; i < waves; ++i) {
    before += part[i][0], tiles_before += part[i][1];
    at += i < wave ? of_wave[i] : 0;
  }
  if (tid == 0) {
    begin[e] = before, tiles[e] = tiles_before;
    if (e == E) begin[E + 1] = pairs, tiles[E + 1] = tiles_before + (count[E] + rows - 1) / rows;
  }
  at += before;
  for (int s = 0; s < steps; ++s) {
    const int p = first + s * 64 + lane;
    bool hit = false;
    if (p < pairs) {
      const int id = ids[p];
      hit = ((uint32_t)id < (uint32_t)E ? id : E) == e;
    }
    const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
    if (hit) order[at + __builtin_popcountll(hits & (((uint64_t)1 << lane) - 1))] = p;
    at += __builtin_popcountll(hits);
  }
}

template <typename T>
struct MmaOf;
template <>
struct MmaOf<half_t> {
  typedef MmaF16 type;
};
template <>
struct MmaOf<bf16_t> {
  typedef MmaBF16 type;
};

struct ExpertArgs {
  const void* X;         // activations: [M, K] (gate / up) or [pairs, K] (down)
  const uint8_t* Wp;     // [E, rows of an expert, K / 2]
  const void* scales;    // [E, rows of an expert, K / group] or null
  const void* zeros;     // the same, or null
  const float* weights;  // down: [pairs]
  void* out;             // gate / up: h [pairs, N]; down: fp32 [pairs, N]
  const int32_t *begin, *tiles, *order;
  int E, top_k, N, K, group, n_blocks;
  float zero_scalar;
};

__device__ __forceinline__ float silu(float x) { return x / (1.0f + __expf(-x)); }

// Tiles of 64 pairs x 64 outputs; a wavefront has 16 outputs (gate / up: 16 gate and 16 up rows).  Per step of 128 values of K the
// activations pass through LDS, the packed weights go from memory to the operand registers: lane (row r16, q) takes the 16 bytes
// with the values 32 q .. 32 q + 31 of the step of its weight row, and at MFMA k-step j the word 4 q + j; the activation operand
// of lane (m = r16, q) holds the same eight k.  K % 32 == 0: such 16 bytes lie inside a row or behind it.
constexpr int kRows = 64, kOuts = 64, kPitch = 128 + 8;

template <typename T, bool UP>
__global__ __launch_bounds__(256) void moe_w4a16_kernel(const ExpertArgs a) {
  typedef typename MmaOf<T>::type Mma;
  constexpr int MT = kRows / 16, NP = UP ? 2 : 1;
  __shared__ __align__(16) T tile[kRows][kPitch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q = lane >> 4;
  const int t = (int)(blockIdx.x / (uint32_t)a.n_blocks);
  if (t >= a.tiles[a.E + (UP ? 1 : 0)]) return;
  int e = 0;
  {
    int lo = 0, hi = a.E;  // the last expert whose tiles begin at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.tiles[mid] <= t) lo = mid; else hi = mid - 1;
    }
    e = lo;
  }
  const int row0 = a.begin[e] + (t - a.tiles[e]) * kRows;
  const int left = a.begin[e + 1] - row0, rows = left < kRows ? left : kRows;
  const int n0 = (int)(blockIdx.x % (uint32_t)a.n_blocks) * kOuts;
  if (UP && e == a.E) {  // pairs without an expert
    T* const h = (T*)a.out;
    for (int i = tid; i < rows * kOuts; i += 256) {
      const int n = n0 + i % kOuts;
      if (n < a.N) h[(int64_t)a.order[row0 + i / kOuts] * a.N + n] = from_float<T>(0.0f);
    }
    return;
  }
  const int groups = a.K / a.group;
  const int n = n0 + wave * 16 + r16;  // this lane's weight row (gate / up: its gate row)
  const int nc = n < a.N ? n : a.N - 1;
  int64_t w_row[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) w_row[i] = (int64_t)e * (NP * a.N) + (int64_t)i * a.N + nc;
  // activation rows: thread tid copies 16-byte chunk tid % 16 of rows tid / 16 + 16 i
  const T* src[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = i * 16 + (tid >> 4);
    const int pair = a.order[row0 + (r < rows ? r : 0)];
    src[i] = (const T*)a.X + (int64_t)(UP ? pair / a.top_k : pair) * a.K;
  }
  const NibbleMagic mg = make_nibble_magic();
  const T one = from_float<T>(1.0f), zs = from_float<T>(a.zero_scalar);
  float4_t acc[NP][MT];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[i][mt] = float4_t{0, 0, 0, 0};

  for (int k0 = 0; k0 < a.K; k0 += 128) {
    const int ka = k0 + (tid & 15) * 8;
    uint4_t v[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) v[i] = ka < a.K ? *(const uint4_t*)(src[i] + ka) : uint4_t{0, 0, 0, 0};
    const int kw = k0 + 32 * q;
    const bool in = kw < a.K;
    uint4_t w[NP];
    T s[NP], z[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      w[i] = in ? *(const uint4_t*)(a.Wp + w_row[i] * (a.K / 2) + kw / 2) : uint4_t{0, 0, 0, 0};
      const int64_t g = w_row[i] * groups + (in ? kw / a.group : 0);
      s[i] = !in ? from_float<T>(0.0f) : a.scales ? ((const T*)a.scales)[g] : one;
      z[i] = !in ? from_float<T>(0.0f) : a.zeros ? ((const T*)a.zeros)[g] : zs;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) *(uint4_t*)&tile[i * 16 + (tid >> 4)][(tid & 15) * 8] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Expand8<T, false> ex(s[i], z[i], mg);
      const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4_t wo = ex(words[j]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[i][mt] = Mma::mma(wo, *(const uint4_t*)&tile[mt * 16 + r16][32 * q + 8 * j], acc[i][mt]);
      }
    }
  }
  // lane (r16, q) holds rows m = 16 mt + r16, outputs 4 q .. 4 q + 3 of the wavefront's 16 (N % 16 == 0: all inside or all outside)
  const int no = n0 + wave * 16 + 4 * q;
  if (no >= a.N) return;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = mt * 16 + r16;
    if (r >= rows) continue;
    const int pair = a.order[row0 + r];
    if (UP) {
      T o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = from_float<T>(silu(acc[0][mt][i]) * acc[NP - 1][mt][i]);
      *(uint2_t*)((T*)a.out + (int64_t)pair * a.N + no) = bitcast<uint2_t>(o);
    } else {
      *(float4_t*)((float*)a.out + (int64_t)pair * a.N + no) = acc[0][mt] * a.weights[pair];
    }
  }
}

// y[t] = the sum of token t's rows, slot by slot
__global__ __launch_bounds__(256) void moe_combine_kernel(const float* __restrict__ rows, const int32_t* __restrict__ ids, void* __restrict__ Y,
                                                         int64_t quads, int N4, int top_k, int E, int out_dtype) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const int64_t t = i / N4;
  const int n = (int)(i - t * N4) * 4;
  float4_t sum{0, 0, 0, 0};
  for (int j = 0; j < top_k; ++j) {
    if ((uint32_t)ids[t * top_k + j] >= (uint32_t)E) continue;  // (no row was written for it)
    sum += *(const float4_t*)(rows + (t * top_k + j) * (int64_t)N4 * 4 + n);
  }
  const int64_t o = t * N4 * 4 + n;
  if (out_dtype == TLQ_F32) {
    *(float4_t*)((float*)Y + o) = sum;
  } else if (out_dtype == TLQ_F16) {
    const half_t h[4] = {(half_t)sum[0], (half_t)sum[1], (half_t)sum[2], (half_t)sum[3]};
    *(uint2_t*)((half_t*)Y + o) = bitcast<uint2_t>(h);
  } else {
    *(uint2_t*)((uint16_t*)Y + o) = uint2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

// tiles of `rows` pairs that E experts (and the pairs without one) can need at most
int64_t most_tiles(int64_t pairs, int64_t E, int64_t rows) {
  const int64_t some = pairs < E + 1 ? pairs : E + 1;
  return some + (pairs - some) / rows;
}

int check_experts(const char* what, int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K, int64_t group, int dtype) {
  TLQ_REQUIRE(M >= 0 && E >= 1 && E <= kMaxExperts && top_k >= 1 && top_k <= 64, "%s: bad shape M=%lld E=%lld top_k=%lld (at most 1024 experts, 64 of them for a token)",
              what, (long long)M, (long long)E, (long long)top_k);
  TLQ_REQUIRE(M * top_k < ((int64_t)1 << 24), "%s: M * top_k = %lld is 2^24 or more: call it for fewer tokens at once", what, (long long)(M * top_k));
  TLQ_REQUIRE(N >= 16 && N % 16 == 0 && N < ((int64_t)1 << 24), "%s: N=%lld must be a multiple of 16", what, (long long)N);
  TLQ_REQUIRE(K >= 32 && K % 32 == 0 && K < ((int64_t)1 << 24), "%s: K=%lld must be a multiple of 32", what, (long long)K);
  TLQ_REQUIRE(group >= 32 && group % 32 == 0 && K % group == 0, "%s: group=%lld must be a multiple of 32 that divides K=%lld", what,
              (long long)group, (long long)K);
  TLQ_REQUIRE(dtype == TLQ_F16 || dtype == TLQ_BF16, "%s: in_dtype must be float16 or bfloat16 (got %d)", what, dtype);
  return 0;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <bool UP>
int run_experts(const char* what, ExpertArgs a, const void* ids, int64_t pairs, int dtype, void* ws, hipStream_t st) {
  const PlanPtrs p = plan_at(ws, a.E);
  a.begin = p.begin, a.tiles = p.tiles, a.order = p.order;
  moe_plan_kernel<<<a.E + 1, kPlanThreads, 0, st>>>((const int32_t*)ids, p.begin, p.tiles, p.order, (int)pairs, a.E, kRows);
  if (!check_launch(what, "moe_plan_kernel")) return 1;
  a.n_blocks = (int)ceil_div((int64_t)a.N, (int64_t)kOuts);
  const int64_t grid = most_tiles(pairs, a.E, kRows) * a.n_blocks;
  TLQ_REQUIRE(grid < ((int64_t)1 << 31), "%s: %lld work-groups: call it for fewer tokens at once", what, (long long)grid);
  if (dtype == TLQ_F16)
    moe_w4a16_kernel<half_t, UP><<<(unsigned)grid, 256, 0, st>>>(a);
  else
    moe_w4a16_kernel<bf16_t, UP><<<(unsigned)grid, 256, 0, st>>>(a);
  return check_launch(what, "moe_w4a16_kernel") ? 0 : 1;
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int64_t tlq_moe_gate_up_workspace_bytes(int64_t M, int64_t E, int64_t top_k) {
  if (M <= 0 || E < 1 || top_k < 1 || E > kMaxExperts || top_k > 64 || M >= ((int64_t)1 << 24)) return 0;
  return plan_bytes(E, M * top_k);
}

extern "C" int64_t tlq_moe_down_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t N) {
  const int64_t plan = tlq_moe_gate_up_workspace_bytes(M, E, top_k);
  if (plan == 0 || N < 1 || N >= ((int64_t)1 << 24)) return 0;
  return plan + M * top_k * N * 4;
}

extern "C" int tlq_moe_gate_up_w4a16(const void* X, const void* ids, const void* w_packed, const void* scales, const void* zeros, void* H,
                                     void* workspace, int64_t workspace_bytes, int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K,
                                     int64_t group, float zero_scalar, int dtype, void* stream) {
  const char* const what = "tlq_moe_gate_up_w4a16";
  if (check_experts(what, M, E, top_k, N, K, group, dtype)) return 1;
  if (M == 0) return 0;
  TLQ_REQUIRE(X && ids && w_packed && H, "%s: null pointer", what);
  TLQ_REQUIRE(aligned16(X) && aligned16(w_packed) && aligned16(H) && ((uintptr_t)ids & 3) == 0 && (((uintptr_t)scales | (uintptr_t)zeros) & 1) == 0,
              "%s: X, w_packed and H must be 16-byte aligned, the others to their type", what);
  const int64_t want = tlq_moe_gate_up_workspace_bytes(M, E, top_k);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && aligned16(workspace), "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  ExpertArgs a{X, (const uint8_t*)w_packed, scales, zeros, nullptr, H, nullptr, nullptr, nullptr, (int)E, (int)top_k, (int)N, (int)K, (int)group, 0, zero_scalar};
  return run_experts<true>(what, a, ids, M * top_k, dtype, workspace, (hipStream_t)stream);
}

extern "C" int tlq_moe_down_w4a16(const void* H, const void* ids, const void* weights, const void* w_packed, const void* scales,
                                  const void* zeros, void* Y, void* workspace, int64_t workspace_bytes, int64_t M, int64_t E, int64_t top_k,
                                  int64_t N, int64_t K, int64_t group, float zero_scalar, int in_dtype, int out_dtype, void* stream) {
  const char* const what = "tlq_moe_down_w4a16";
  if (check_experts(what, M, E, top_k, N, K, group, in_dtype)) return 1;
  TLQ_REQUIRE(out_dtype == TLQ_F16 || out_dtype == TLQ_BF16 || out_dtype == TLQ_F32, "%s: out_dtype must be float16, bfloat16 or float32 (got %d)", what, out_dtype);
  if (M == 0) return 0;
  TLQ_REQUIRE(H && ids && weights && w_packed && Y, "%s: null pointer", what);
  TLQ_REQUIRE(aligned16(H) && aligned16(w_packed) && aligned16(Y) && (((uintptr_t)ids | (uintptr_t)weights) & 3) == 0 && (((uintptr_t)scales | (uintptr_t)zeros) & 1) == 0,
              "%s: H, w_packed and Y must be 16-byte aligned, the others to their type", what);
  const int64_t want = tlq_moe_down_workspace_bytes(M, E, top_k, N);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && aligned16(workspace), "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  const int64_t pairs = M * top_k;
  float* const rows = (float*)((uint8_t*)workspace + plan_bytes(E, pairs));
  ExpertArgs a{H, (const uint8_t*)w_packed, scales, zeros, (const float*)weights, rows, nullptr, nullptr, nullptr, (int)E, (int)top_k, (int)N, (int)K, (int)group, 0, zero_scalar};
  hipStream_t st = (hipStream_t)stream;
  if (run_experts<false>(what, a, ids, pairs, in_dtype, workspace, st)) return 1;
  const int64_t quads = M * (N / 4);
  moe_combine_kernel<<<(unsigned)ceil_div(quads, (int64_t)256), 256, 0, st>>>(rows, (const int32_t*)ids, Y, quads, (int)(N / 4), (int)top_k, (int)E, out_dtype);
  return check_launch(what, "moe_combine_kernel") ? 0 : 1;
}
