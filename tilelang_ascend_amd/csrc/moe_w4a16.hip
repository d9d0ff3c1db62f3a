// The experts' products of a mixture-of-experts layer on packed 4-bit weights.
//   gate / up:  h[t, j, n] = silu(x[t] . W[e, n]) * (x[t] . W[e, N + n]),  e = ids[t, j]
//   down:       y[t, n] = sum_j w[t, j] * (h[t, j] . W[e, n])
// W = rn_T(rn_T(T(u) - z) * s) as everywhere in this library, fp32 sums.  A pair (t, j) whose id names no expert has h = 0 and
// adds nothing.
//
// Pairs are sorted by expert first (moe_plan_kernel: counts, where each expert's pairs begin, the pairs in order -- a pair keeps
// its place among those of its expert, so nothing depends on timing), then every expert's rows are cut into tiles of activation
// rows, which work-groups find by their number.
#include <type_traits>

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

// ---- few pairs: weights resident in registers -----------------------------------------------------------------------------
// A wavefront asks for all its packed weights at once -- 16 weight rows x up to BPW blocks of 128 values of K, 1 KB a block -- and
// keeps them while it multiplies them with the expert's pairs, `row_cap` of them a pass.  Every weight is read once whatever the
// number of pairs, a CU has some 64 - 128 KB in flight, and no launch sorts the pairs first: a work-group looks its expert's pairs
// up among all ids (at most kFewPairs).  The work-groups of an expert are those of the first pair that names it, or, where there
// are more pairs than experts, those of the expert's number; one token's pairs are taken one by one.
//   A tile is 16 weight rows: 16 outputs, or 8 gate rows and the 8 up rows that go with them.  A work-group has `tiles` of them side by
// side, each shared by `splits` wavefronts that take a part of K each; their sums meet in LDS and are added in the order of K.
//   Activations (a pass's rows, whole), scales and zero points of the tiles go global -> LDS ahead of the weights and are waited
// for by count, with the weights still on their way.
constexpr int kFewPairs = 2048;
enum { kFewByPair = 1, kFewOneToken = 2, kFewFold = 4 };

struct FewArgs {
  const void* X;
  const uint8_t* Wp;
  const void* scales;
  const void* zeros;
  const float* weights;
  const int32_t* ids;
  void* out;
  int pairs, E, top_k, N, K, groups;
  uint32_t per_group;  // ceil(2^32 / (group / 32)), 0 for groups of 32
  float zero_scalar;
  int n_groups;                            // work-groups of an expert
  uint32_t shape;                          // tiles | splits << 8 | row_cap << 16 | flags << 24 (kFewFold: the scalar zero point is a small integer)
};

__device__ __forceinline__ bool small_integer(float z) { return z == __builtin_rintf(z) && z >= -256.0f && z <= 256.0f; }

// 16 bytes per lane, global -> LDS: lane l to lds + 16 l (lanes that are switched off: nothing)
__device__ __forceinline__ void direct16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}
template <typename T, bool UP, int BPW>
__global__ __launch_bounds__(512, 2) void moe_few_kernel(const FewArgs a) {
  typedef typename MmaOf<T>::type Mma;
  typedef __attribute__((address_space(3))) uint8_t* lptr_t;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tiles = a.shape & 255, splits = (a.shape >> 8) & 255, row_cap = (a.shape >> 16) & 255, flags = a.shape >> 24;
  const int waves = tiles * splits, threads = waves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
  const int who = (int)(blockIdx.x / (uint32_t)a.n_groups), group_no = (int)blockIdx.x - who * a.n_groups;
  const bool by_pair = flags & kFewByPair, one_token = flags & kFewOneToken;
  const int blocks = (a.K + 127) >> 7, groups = a.groups;
  const int pitch = blocks * 256 + 16;  // bytes of an activation row: 16 more, so that the rows of an operand lie on different banks
  // LDS: activation rows, scales, zero points, sums of the other wavefronts, the pairs
  uint8_t* const act = smem;
  const uint32_t act_lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)smem);
  const int sc_at = row_cap * pitch, zp_at = sc_at + (a.scales ? tiles * 32 * groups : 0), sums_at = zp_at + (a.zeros ? tiles * 32 * groups : 0);
  float* const sums = (float*)(smem + sums_at);
  int32_t* const head = (int32_t*)(sums + tiles * (splits - 1) * 256);  // [0] number of pairs, [1] an earlier pair has this expert
  uint16_t* const list = (uint16_t*)(head + 4);

  const int e = by_pair ? __builtin_amdgcn_readfirstlane(a.ids[who]) : who;
  const bool none = (uint32_t)e >= (uint32_t)a.E;
  constexpr int OUTS = UP ? 8 : 16;  // outputs of a tile
  const int n_tiles = a.N / OUTS, tile0 = group_no * tiles;
  if (none && (!UP || by_pair)) {
    if (!UP) return;
    T* const h = (T*)a.out + (int64_t)who * a.N;
    const int end = (tile0 + tiles) * OUTS;
    for (int n = tile0 * OUTS + tid; n < end && n < a.N; n += threads) h[n] = from_float<T>(0.0f);
    return;
  }

  // the expert's pairs
  int count = 1;
  if (one_token) {
    if (tid == 0) list[0] = (uint16_t)who;  // (read behind the barrier that the rows are waited for at)
  } else {
    if (tid < 2) head[tid] = 0;
    __syncthreads();
    for (int p = tid; p < a.pairs; p += threads) {
      const int id = a.ids[p];
      if (none ? (uint32_t)id >= (uint32_t)a.E : id == e) {
        if (by_pair && p < who) head[1] = 1;
        list[atomicAdd(&head[0], 1)] = (uint16_t)p;
      }
    }
    __syncthreads();
    count = __builtin_amdgcn_readfirstlane(head[0]);
    if (count == 0 || (by_pair && __builtin_amdgcn_readfirstlane(head[1]))) return;
  }
  if (UP && none) {
    T* const h = (T*)a.out;
    const int width = tiles * OUTS;
    for (int i = tid; i < count * width; i += threads) {
      const int n = tile0 * OUTS + i % width;
      if (n < a.N) h[(int64_t)list[i / width] * a.N + n] = from_float<T>(0.0f);
    }
    return;
  }

  // a pass's rows -> LDS; and zeros up to the end of the last block
  auto load_rows = [&](int row0, int rows) __attribute__((always_inline)) {
    for (int r = wave; r < rows; r += waves) {
      const int pair = one_token ? who : __builtin_amdgcn_readfirstlane((int)list[row0 + r]);
      const uint8_t* const x = (const uint8_t*)((const T*)a.X + (int64_t)(UP ? pair / a.top_k : pair) * a.K);
      for (int at = 0; at < a.K * 2; at += 1024)
        if (at + lane * 16 < a.K * 2) direct16(x + at + lane * 16, act_lds + r * pitch + at);
      if (a.K * 2 + lane * 16 < blocks * 256) *(uint4_t*)(act + r * pitch + a.K * 2 + lane * 16) = uint4_t{0, 0, 0, 0};
    }
  };
  // scales and zero points: half tiles of 8 rows, back to back in memory and in LDS (16 * groups bytes each)
  const int chunks = tiles * 2 * groups;
  auto group_values = [&](int c) -> int64_t {  // where the eight values of chunk c lie in their tensors
    const int half = c / groups, at = c - half * groups;
    int t = tile0 + (half >> 1);
    t = t < n_tiles ? t : n_tiles - 1;
    const int64_t row = UP ? (int64_t)e * 2 * a.N + (half & 1) * a.N + t * 8 : (int64_t)e * a.N + t * 16 + (half & 1) * 8;
    return row * groups + at * 8;
  };
  // (nothing is on its way here or behind the loop below; said so, because the compiler would wait once more, for the direct loads)
  const auto nothing_on_its_way = []() __attribute__((always_inline)) { __builtin_amdgcn_s_waitcnt(0x0f70); };
  nothing_on_its_way();
  if ((((uintptr_t)a.scales | (uintptr_t)a.zeros) & 15) == 0) {
    load_rows(0, count < row_cap ? count : row_cap);
    for (int c0 = wave * 64; c0 < chunks; c0 += threads) {
      if (c0 + lane >= chunks) continue;
      const int64_t off = group_values(c0 + lane);
      if (a.scales) direct16((const T*)a.scales + off, act_lds + sc_at + c0 * 16);
      if (a.zeros) direct16((const T*)a.zeros + off, act_lds + zp_at + c0 * 16);
    }
  } else {  // value by value; ahead of the rows, because loads into registers wait for everything before them
    for (int i = tid; i < chunks * 8; i += threads) {
      const int64_t off = group_values(i >> 3) + (i & 7);
      if (a.scales) ((T*)(smem + sc_at))[i] = ((const T*)a.scales)[off];
      if (a.zeros) ((T*)(smem + zp_at))[i] = ((const T*)a.zeros)[off];
    }
    nothing_on_its_way();
    load_rows(0, count < row_cap ? count : row_cap);
  }
  // the weights: lane (r16, q) takes the 32 values 32 q .. of every block of row r16
  const int my_tile = wave / splits, split = wave - my_tile * splits;
  const int tile = tile0 + my_tile < n_tiles ? tile0 + my_tile : n_tiles - 1;
  const int per = (blocks + splits - 1) / splits, block0 = split * per;
  const int mine = blocks - block0 < per ? (blocks - block0 < 0 ? 0 : blocks - block0) : per;
  uint4_t w[BPW];
  {
    const int64_t row = UP ? (int64_t)e * 2 * a.N + (r16 >> 3) * a.N + tile * 8 + (r16 & 7) : (int64_t)e * a.N + tile * 16 + r16;
    // BPW loads whatever there is to load, so that they can be counted: past the end, an address of the row that is asked for anyway
    // (behind K the rows in LDS are zeros)
    const uint8_t* const src = a.Wp + row * (a.K / 2);
    const int off = (mine > 0 ? block0 : 0) * 64 + q * 16, last = a.K / 2 - 16;
#pragma unroll
    for (int b = 0; b < BPW; ++b) {
      const int at = b < mine ? off + b * 64 : off;
      w[b] = __builtin_nontemporal_load((const uint4_t*)(src + (at < last ? at : last)));
    }
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(BPW) : "memory");  // all but the weights
  __syncthreads();

  const NibbleMagic mg = make_nibble_magic();
  const T one = from_float<T>(1.0f), zs = from_float<T>(a.zero_scalar);
  const T* const my_sc = (const T*)(smem + sc_at) + (my_tile * 16 + r16) * groups;
  const T* const my_zp = (const T*)(smem + zp_at) + (my_tile * 16 + r16) * groups;
  bool fold = flags & kFewFold;
  if (a.zeros) {  // are this tile's zero points small integers?
    bool ok = true;
    for (int c = lane; c < 2 * groups; c += 64) {
      const uint4_t v = *(const uint4_t*)(smem + zp_at + (my_tile * 2 * groups + c) * 16);
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) ok = ok && small_integer(to_float(bitcast<T>((uint16_t)x[i]))) && small_integer(to_float(bitcast<T>((uint16_t)(x[i] >> 16))));
    }
    fold = __builtin_amdgcn_ballot_w64(ok) == ~0ull;
  }

  auto pass = [&](int row0, int rows) __attribute__((always_inline)) {
    float4_t acc[2] = {float4_t{0, 0, 0, 0}, float4_t{0, 0, 0, 0}};
    const uint8_t* const my_act = act + (r16 < rows ? r16 : rows - 1) * pitch + q * 64 + block0 * 256;
    auto multiply = [&](auto fold_tag) __attribute__((always_inline)) {
      constexpr bool FOLD = decltype(fold_tag)::value;
#pragma unroll
      for (int b = 0; b < BPW; ++b) {
        if (b >= mine) break;
        const uint32_t u = (uint32_t)((block0 + b) * 4 + q), at = a.per_group ? __umulhi(u, a.per_group) : u;
        const uint32_t g = (int)at < groups ? at : groups - 1;  // (behind K, where the rows hold zeros)
        const Expand8<T, FOLD> ex(a.scales ? my_sc[g] : one, a.zeros ? my_zp[g] : zs, mg);
        // (opaque: the expanded weights are the same in every pass, and would be kept, four times as many registers as there are)
        asm volatile("" : "+v"(w[b].x), "+v"(w[b].y), "+v"(w[b].z), "+v"(w[b].w));
        const uint32_t words[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j & 1] = Mma::mma(ex(words[j]), *(const uint4_t*)(my_act + b * 256 + j * 16), acc[j & 1]);
      }
    };
    if (fold) multiply(std::true_type{});
    else multiply(std::false_type{});
    float4_t sum = acc[0] + acc[1];
    if (splits > 1) {
      if (split) *(float4_t*)(sums + ((my_tile * (splits - 1) + split - 1) * 64 + lane) * 4) = sum;
      __syncthreads();
      if (split) return;
      for (int i = 1; i < splits; ++i) sum += *(const float4_t*)(sums + ((my_tile * (splits - 1) + i - 1) * 64 + lane) * 4);
    }
    // lane (r16, q): outputs 4 q .. 4 q + 3 of pair r16; gate / up: gates in q = 0, 1, their ups 32 lanes on
    const bool live = r16 < rows && tile0 + my_tile < n_tiles;
    if constexpr (UP) {
      float4_t up;
#pragma unroll
      for (int i = 0; i < 4; ++i) up[i] = __shfl_xor(sum[i], 32);
      if (q < 2 && live) {
        T o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = from_float<T>(silu(sum[i]) * up[i]);
        *(uint2_t*)((T*)a.out + (int64_t)list[row0 + r16] * a.N + tile * 8 + q * 4) = bitcast<uint2_t>(o);
      }
    } else if (live) {
      const int pair = list[row0 + r16];
      *(float4_t*)((float*)a.out + (int64_t)pair * a.N + tile * 16 + q * 4) = sum * a.weights[pair];
    }
  };
  // (the first pass apart from the loop: ahead of a loop the compiler waits for all weights, and here they are to be waited for one by one)
  pass(0, count < row_cap ? count : row_cap);
  for (int row0 = row_cap; row0 < count; row0 += row_cap) {
    const int rows = count - row0 < row_cap ? count - row0 : row_cap;
    __syncthreads();  // (the last pass's rows have been read, its sums added up)
    load_rows(row0, rows);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    pass(row0, rows);
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

// How moe_few_kernel is launched.  ok: it takes the call.
struct FewPlan {
  bool ok;
  int tiles, splits, bpw, row_cap, n_groups;
  bool by_pair;
  int64_t lds, blocks;
};
FewPlan few_plan(bool up, int64_t pairs, int64_t E, int64_t N, int64_t K, int64_t group, bool scales, bool zeros) {
  FewPlan p{};
  const int64_t blocks = ceil_div(K, (int64_t)128), n_tiles = N / (up ? 8 : 16), groups = K / group;
  const int64_t experts = pairs < E ? pairs : E;
  if (pairs > kFewPairs || pairs > experts * 8 || blocks > 8 * 16) return p;
  p.splits = 1;
  while (ceil_div(blocks, (int64_t)p.splits) > 16) p.splits *= 2;
  while (p.splits < 8 && p.splits * 2 <= blocks && experts * n_tiles * p.splits < 2048) p.splits *= 2;
  const int64_t per = ceil_div(blocks, (int64_t)p.splits);
  p.bpw = per <= 4 ? 4 : per <= 8 ? 8 : 16;
  p.tiles = p.splits >= 4 ? 1 : 4 / p.splits;
  p.by_pair = pairs <= E;
  // rows of a pass: twice what an expert has on average, while they leave LDS for two work-groups
  const int64_t pitch = blocks * 256 + 16, average = ceil_div(pairs, experts);
  p.row_cap = 16;
  while (p.row_cap > 1 && (p.row_cap >= 4 * average || p.row_cap * pitch > 60 * 1024)) p.row_cap /= 2;
  p.n_groups = (int)ceil_div(n_tiles, (int64_t)p.tiles);
  p.lds = p.row_cap * pitch + (int64_t)((scales ? 1 : 0) + (zeros ? 1 : 0)) * p.tiles * 16 * groups * 2 + (int64_t)p.tiles * (p.splits - 1) * 1024 + 16 + ceil_div(pairs, (int64_t)8) * 16;
  p.blocks = (p.by_pair ? pairs : E + (up ? 1 : 0)) * p.n_groups;
  p.ok = p.lds <= 160 * 1024 && p.blocks < ((int64_t)1 << 31);
  return p;
}

template <typename T, bool UP, int BPW>
int launch_few(const char* what, const FewArgs& a, const FewPlan& p, hipStream_t st) {
  auto kern = moe_few_kernel<T, UP, BPW>;
  static bool attr_set = false;
  if (!attr_set) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    TLQ_REQUIRE(e == hipSuccess, "%s: cannot reserve LDS: %s", what, hipGetErrorString(e));
    attr_set = true;
  }
  kern<<<(unsigned)p.blocks, p.tiles * p.splits * 64, (size_t)p.lds, st>>>(a);
  return check_launch(what, "moe_few_kernel") ? 0 : 1;
}

template <bool UP>
int run_few(const char* what, const ExpertArgs& x, const void* ids, int64_t pairs, int dtype, const FewPlan& p, hipStream_t st) {
  const bool whole = x.zero_scalar == (float)(int)x.zero_scalar && x.zero_scalar >= -256.0f && x.zero_scalar <= 256.0f;
  const int units = x.group / 32;
  const int flags = (p.by_pair ? kFewByPair : 0) | (p.by_pair && pairs == x.top_k ? kFewOneToken : 0) | (whole ? kFewFold : 0);
  const FewArgs a{x.X, x.Wp, x.scales, x.zeros, x.weights, (const int32_t*)ids, x.out, (int)pairs, x.E, x.top_k, x.N, x.K, x.K / x.group,
                  units == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + units - 1) / units), x.zero_scalar, p.n_groups,
                  (uint32_t)(p.tiles | p.splits << 8 | p.row_cap << 16 | flags << 24)};
#define TLQ_FEW(BPW) (dtype == TLQ_F16 ? launch_few<half_t, UP, BPW>(what, a, p, st) : launch_few<bf16_t, UP, BPW>(what, a, p, st))
  return p.bpw == 4 ? TLQ_FEW(4) : p.bpw == 8 ? TLQ_FEW(8) : TLQ_FEW(16);
#undef TLQ_FEW
}

template <bool UP>
int run_experts(const char* what, ExpertArgs a, const void* ids, int64_t pairs, int dtype, void* ws, hipStream_t st) {
  const FewPlan few = few_plan(UP, pairs, a.E, a.N, a.K, a.group, a.scales != nullptr, a.zeros != nullptr);
  if (few.ok) return run_few<UP>(what, a, ids, pairs, dtype, few, st);
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
