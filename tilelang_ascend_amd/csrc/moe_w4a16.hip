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

#include "moe.h"

namespace tlq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxExperts = 1024;

// The plan in the workspace: how many tiles there are, the pairs by expert, tiles of few pairs, tiles of 256 pairs.  With tiles of 256 pairs
// (with_large: the work-groups of one of them, 0: none) an expert's last tile is one of them if it has `from` pairs, and tiles of 64 pairs take
// what is left otherwise.
//   Up to kCompactPairs pairs the work-groups of the plan know the counts of all experts.  Tiles follow each other, and `from` is chosen for
// the fewest rounds of work-groups (choose_from).  With more pairs a tile's place goes by the pairs before it alone -- tiles of `rows` pairs of
// expert e begin at place (pairs before e) / rows + e, what is left beside large tiles at e --, which leaves at most one place an expert empty;
// `from` is 65, and beside large tiles the pairs without an expert are cut into kNoneTiles tiles at most (places for all pairs in tiles of 64
// would be work-groups that find nothing to do).
constexpr int kCompactPairs = 4096, kNoneTiles = 64, kLargeFrom = 65;
__host__ __device__ inline int large_tiles(int pairs, int from) { return pairs + kLargeRows <= from ? 0 : (pairs + kLargeRows - from) / kLargeRows; }
struct PlanSizes {
  int64_t small, large;  // places for tiles
};
inline PlanSizes plan_sizes(int64_t E, int64_t pairs, int64_t rows, bool large) {
  const int64_t some = pairs < E + 1 ? pairs : E + 1;
  PlanSizes z;
  z.small = pairs > kCompactPairs ? pairs / rows + E + 1 : some + (pairs - some) / rows;
  if (large && pairs > kCompactPairs) z.small = E + kNoneTiles;
  z.large = !large ? 0 : pairs > kCompactPairs ? pairs / kLargeRows + E : pairs / kLargeFrom;
  return z;
}
inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
struct PlanPtrs {
  int32_t *totals, *order;
  PlanTile *small, *large;
};
inline PlanPtrs plan_at(void* ws, int64_t pairs, const PlanSizes& z) {
  uint8_t* const p = (uint8_t*)ws + 256;
  uint8_t* const small = p + align256(pairs * 4);
  return {(int32_t*)ws, (int32_t*)p, (PlanTile*)small, (PlanTile*)(small + align256(z.small * 16))};
}
inline int64_t plan_bytes_of(int64_t E, int64_t pairs, int64_t rows, bool large) {
  const PlanSizes z = plan_sizes(E, pairs, rows, large);
  return 256 + align256(pairs * 4) + align256(z.small * 16) + align256(z.large * 16);
}
inline int64_t plan_bytes(int64_t E, int64_t pairs) {  // of these pairs and of fewer
  const int64_t a = plan_bytes_of(E, pairs, 32, false), b = plan_bytes_of(E, pairs, 64, false), c = plan_bytes_of(E, pairs, 64, true);
  const int64_t most = a > b ? (a > c ? a : c) : (b > c ? b : c), fewer = pairs > kCompactPairs ? plan_bytes(E, kCompactPairs) : 0;
  return most > fewer ? most : fewer;
}

// Candidates for `from`: 65, 129, 193, 256 (whole tiles only), and more pairs than there are (none).  A round of large tiles is 256 work-groups,
// one a CU; of tiles of 64 pairs as wide as those 512 go at once and take 5 / 8 of its time (gate / up, 16 experts of 2048 x 4096: 98 and 61 us).
constexpr int kFromChoices = 5;
__device__ __forceinline__ int from_choice(int i) { return i < 3 ? 64 * i + 65 : i == 3 ? kLargeRows : 1 << 24; }
__device__ __forceinline__ int rounds_of(int large, int small, int groups) { return 8 * ((large * groups + 255) / 256) + 5 * ((small * groups + 511) / 512); }

// One work-group per expert, and one more for the pairs without one: each looks at all pairs and writes down its own.  A wavefront takes
// a run of pairs, so that a pair's place is that of its wavefront, its step and its lane; sixteen steps' ids are asked for at once (65536 pairs of 64
// experts: one by one, with an LDS histogram of all experts, 44 us).  Up to 1024 pairs 256 threads, which come and go faster (layer of 16 tokens on 8 of
// 256 experts of 1024 x 4096: 180 -> 174 us for two plans; 128 tokens on 8 of 512 of 512 x 1024, gate / up 50 -> 45).
template <bool COMPACT, int THREADS>
__global__ __launch_bounds__(THREADS) void moe_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ totals,
                                                               int32_t* __restrict__ order, PlanTile* __restrict__ small,
                                                               PlanTile* __restrict__ large, int pairs, int E, int rows, int with_large) {
  constexpr int waves = THREADS / 64, AHEAD = COMPACT ? 4 : 16;
  __shared__ int32_t count[COMPACT ? kMaxExperts + 1 : 1];
  __shared__ int32_t part[waves][4];
  __shared__ int32_t tiles_of[kFromChoices][2];  // large and small tiles that each choice makes
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = blockIdx.x;
  if (COMPACT) {
    for (int i = tid; i <= E; i += THREADS) count[i] = 0;
    if (tid < 2 * kFromChoices) tiles_of[tid >> 1][tid & 1] = 0;
    __syncthreads();
  }
  const int steps = (pairs + THREADS - 1) / THREADS;
  const int first = wave * steps * 64;
  // f(a pair, its expert or E, whether there is one) for every step of this wavefront
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    for (int s0 = 0; s0 < steps; s0 += AHEAD) {
      int id[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int p = first + (s0 + i) * 64 + lane;
        id[i] = ids[s0 + i < steps && p < pairs ? p : 0];
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int p = first + (s0 + i) * 64 + lane;
        f(p, (uint32_t)id[i] < (uint32_t)E ? id[i] : E, s0 + i < steps && p < pairs);
      }
    }
  };
  int own = 0, fewer = 0;  // pairs of this expert, and of those before it, in the wavefront's run
  each([&](int, int at, bool there) __attribute__((always_inline)) {
    if (COMPACT) {
      if (there) atomicAdd(&count[at], 1);  // (whole numbers: in any order)
    } else {
      fewer += __builtin_popcountll(__builtin_amdgcn_ballot_w64(there && at < e));
    }
    own += __builtin_popcountll(__builtin_amdgcn_ballot_w64(there && at == e));
  });
  int small_before = 0, large_before = 0, from = kLargeFrom;
  if (COMPACT) {
    __syncthreads();
    if (with_large) {  // (the same in every work-group)
      for (int c = 0; c < kFromChoices; ++c) {
        int l = 0, m = 0;
        for (int i = tid; i < E; i += THREADS) {
          const int n = large_tiles(count[i], from_choice(c)), left = count[i] - n * kLargeRows;
          l += n, m += left > 0 ? (left + rows - 1) / rows : 0;
        }
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o), m += __shfl_xor(m, o);
        if (lane == 0 && (l | m)) atomicAdd(&tiles_of[c][0], l), atomicAdd(&tiles_of[c][1], m);
      }
      __syncthreads();
      int best = 0x7fffffff;
      for (int c = 0; c < kFromChoices; ++c) {
        const int rounds = rounds_of(tiles_of[c][0], tiles_of[c][1], with_large);
        if (rounds < best) best = rounds, from = from_choice(c);
      }
    }
    for (int i = tid; i < e; i += THREADS) {
      const int l = with_large ? large_tiles(count[i], from) : 0, left = count[i] - l * kLargeRows;
      fewer += count[i], large_before += l, small_before += left > 0 ? (left + rows - 1) / rows : 0;
    }
    for (int o = 32; o > 0; o >>= 1) fewer += __shfl_xor(fewer, o), small_before += __shfl_xor(small_before, o), large_before += __shfl_xor(large_before, o);
  }
  if (lane == 0) part[wave][0] = own, part[wave][1] = fewer, part[wave][2] = small_before, part[wave][3] = large_before;
  __syncthreads();
  int at = 0, mine = 0;
  fewer = small_before = large_before = 0;
#pragma unroll
  for (int i = 0; i < waves; ++i) {
    at += i < wave ? part[i][0] : 0;
    mine += part[i][0], fewer += part[i][1], small_before += part[i][2], large_before += part[i][3];
  }
  const int my_large = with_large && e < E ? large_tiles(mine, from) : 0, left = mine - my_large * kLargeRows;
  if (!COMPACT && with_large && e == E && rows < (pairs + kNoneTiles - 1) / kNoneTiles) rows = (pairs + kNoneTiles - 1) / kNoneTiles;
  const int my_small = left > 0 ? (left + rows - 1) / rows : 0;
  int small_end = small_before + my_small, large_end = large_before + my_large;
  if (!COMPACT) {
    small_before = with_large ? e : fewer / rows + e;
    small_end = with_large ? (e < E ? e + 1 : E + my_small) : (fewer + mine) / rows + e + 1;
    large_before = fewer / kLargeRows + e;
    large_end = e < E ? (fewer + mine) / kLargeRows + e + 1 : large_before;
  }
  if (with_large) {
    for (int i = tid; i < large_end - large_before; i += THREADS) {
      const int at = i * kLargeRows, n = i < my_large ? (mine - at < kLargeRows ? mine - at : kLargeRows) : 0;
      large[large_before + i] = PlanTile{e, fewer + at, n, 0};
    }
  }
  for (int i = tid; i < small_end - small_before; i += THREADS) {
    const int at = my_large * kLargeRows + i * rows, n = i < my_small ? (mine - at < rows ? mine - at : rows) : 0;
    small[small_before + i] = PlanTile{e, fewer + at, n, 0};
  }
  if (e == E && tid == 0) totals[0] = small_end, totals[1] = large_end;
  at += fewer;
  each([&](int p, int expert, bool there) __attribute__((always_inline)) {
    const uint64_t hits = __builtin_amdgcn_ballot_w64(there && expert == e);
    if (there && expert == e) order[at + __builtin_popcountll(hits & (((uint64_t)1 << lane) - 1))] = p;
    at += __builtin_popcountll(hits);
  });
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

// Global -> LDS without registers: 16 or 4 bytes per lane, lane l to lds + 16 l or 4 l (lanes that are switched off: nothing).
__device__ __forceinline__ void direct16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void direct16_at(uint32_t off, const uint8_t* base, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void direct4(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src) : "memory");
}

// A zero point that is a small integer can be folded into the unpacking's bias.  In bfloat16 that is worth it (gate / up of 64 experts of 1408 x 2048,
// 400 tokens on 6: 75 us, 98 the other way) and a tensor of zero points is looked at block by block; binary16 subtracts two values in one instruction
// and takes the other way always: 80 -> 73 us, with no look at the zero points and registers for four work-groups on a CU.
template <typename T>
constexpr bool kFolds = !std::is_same<T, half_t>::value;

// ---- tiles of many pairs ----------------------------------------------------------------------------------------------------
// Up to 16 MAXMT pairs of one expert x NT tiles of 16 weight rows for each of four wavefronts (a tile: 16 outputs, or 8 gate rows and the 8
// up rows that go with them).  K goes by in steps of KSB blocks of 128 values: the activation rows are gathered global -> LDS into
// two buffers a step ahead, the packed weights go straight into operand registers a step ahead -- lane (r16, q) has the 32 values 32 q ..
// of each block of row r16, at MFMA k-step j the eight of word 4 q + j --, are expanded there and multiplied with all rows: a weight
// is expanded once per 16 MAXMT pairs, an activation operand read once per NT tiles.  One barrier a step.
//   64 pairs: fp16, zero points, 211 tokens on 2 of 8 experts of 14336 x 4096 (gate / up): 240 - 260 us; the vector units issue for
// 60 % of it, the matrix units are busy for 25 %, 1.36 GB come from behind L2: every further tile of an expert reads its rows again.  With 64 rows of W a wavefront in the
// place of 32 (NT = 4) 5 - 10 % slower -- fewer work-groups on a CU, coarser rounds --; with 128 pairs level where experts have 192 pairs and more, 10 - 30 % slower
// below; tiles of an expert side by side on the same weight rows 3 - 6 % faster on matrices of 58 MB, 2 - 8 % slower on small ones.
//   32 pairs: bf16, 48 tokens on 8 of 128 experts of 768 x 2048 (gate / up): 35 - 40 us for 199 MB, the rate of a large copy.
//   Scales and zero points come through LDS in windows of eight groups (whole steps: 8 groups are 256 (group / 32) values), loaded a window
// ahead as the 16-byte pieces of a row that hold them (two, unless rows are whole pieces).  ANY: zero points that need not be small integers (a tensor, or
// such a scalar).
// u / units for u below 2^30: with 2^shift <= units < 2^(shift + 1) and mul = ceil(2^(31 + shift) / units), mul * units is at most units - 1 < 2^(shift + 1)
// more than 2^(31 + shift), so that u * mul / 2^(31 + shift) is less than 2 u / 2^31 / units <= 1 / units above u / units: the same whole number below.
// (One multiplication and one shift, a power of two or not; a reciprocal of 32 bits alone, ceil(2^32 / units), is wrong from units of 65537 on.)
struct GroupOf {
  uint32_t mul;
  int32_t shift;
  __host__ __device__ __forceinline__ int operator()(int u) const { return (int)((uint32_t)(((uint64_t)((uint32_t)u * 2) * mul) >> 32) >> shift); }
};
inline GroupOf make_group_of(int units) {
  GroupOf g{0, 0};
  while ((units >> g.shift) > 1) ++g.shift;
  g.mul = (uint32_t)((((uint64_t)1 << (31 + g.shift)) + units - 1) / units);
  return g;
}

struct TileArgs {
  const void* X;
  const uint8_t* Wp;
  const void* scales;
  const void* zeros;
  const float* weights;  // down: of the pairs
  void* out;             // gate / up: h [pairs, N], or with K in parts fp32 sums [part][pair][2 N]; down: weighted fp32 rows [part][pair][N]
  const PlanTile* tiles;
  const int32_t* order;  // (how many tiles there are: at order[-64])
  int pairs, E, top_k, N, K, groups;
  GroupOf group_of;    // of the u-th 32 values of a row
  float zero_scalar;
  int n_groups;        // work-groups side by side
  int window;          // steps of a window
  int chunk_steps;     // steps of a work-group: those of a part of K (few tiles), whose sums moe_combine_kernel or moe_gate_kernel adds
};

template <int MAXMT, int NT, int KSB>
struct TileCfg {
  static constexpr int ROWS = 16 * MAXMT, ROW_BYTES = KSB * 256, ACT = ROWS * ROW_BYTES;
  static constexpr int TILES = 4 * NT, WINDOW = TILES * 16 * 16;          // scales of a window: a piece of every row, or two
  static constexpr int RPI = 1024 / ROW_BYTES, LOADS = ROWS / RPI / 4;    // rows of a load instruction, loads of a wavefront and step
  static_assert(ROWS % (RPI * 4) == 0, "the rows split over the wavefronts");
  static constexpr int lds(int pieces, bool zeros) { return 2 * ACT + 2 * WINDOW * pieces * (zeros ? 2 : 1); }
};

template <typename T, bool UP, bool ANY, int MAXMT, int NT, int KSB>
__global__ __launch_bounds__(256, ANY && kFolds<T> ? 3 : 4) void moe_tile_kernel(const TileArgs a) {
  typedef typename MmaOf<T>::type Mma;
  typedef TileCfg<MAXMT, NT, KSB> Cfg;
  typedef __attribute__((address_space(3))) uint8_t* lptr_t;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
  // Work-groups of a tile, and tiles of an expert, which follow each other, on one XCD (numbers go to the XCDs in turn): they share
  // activation rows and weights.
  const int all_steps = (a.K + KSB * 128 - 1) / (KSB * 128), chunks = (all_steps + a.chunk_steps - 1) / a.chunk_steps;
  const int live = a.order[-64] * chunks * a.n_groups;
  if ((int)blockIdx.x >= live) return;
  const int no = addr::xcd_order(blockIdx.x, live);
  const int part = (int)((uint32_t)no / (uint32_t)a.n_groups), group_no = no - part * a.n_groups;
  const int tile_no = part / chunks, chunk = part - tile_no * chunks;
  const PlanTile pt = a.tiles[tile_no];
  const int e = __builtin_amdgcn_readfirstlane(pt.expert), first = __builtin_amdgcn_readfirstlane(pt.first), rows = __builtin_amdgcn_readfirstlane(pt.pairs);
  if (rows == 0) return;
  constexpr int OUTS = UP ? 8 : 16;
  const int n_tiles = a.N / OUTS, tile0 = group_no * Cfg::TILES;
  if (e == a.E) {  // pairs without an expert
    if constexpr (UP) {
      if (chunks > 1) return;  // (moe_gate_kernel writes their zeros)
      T* const h = (T*)a.out;
      constexpr int width = Cfg::TILES * OUTS;
      for (int i = tid; i < rows * width; i += 256) {
        const int n = tile0 * OUTS + i % width;
        if (n < a.N) h[(int64_t)a.order[first + i / width] * a.N + n] = from_float<T>(0.0f);
      }
    }
    return;
  }
  const int pieces = a.groups % 8 == 0 ? 1 : 2, window_bytes = Cfg::WINDOW * pieces;
  uint8_t* const sc = smem + 2 * Cfg::ACT;
  uint8_t* const zp = sc + 2 * window_bytes;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)smem);
  const int32_t* const mine = a.order + first;

  // Activation rows: lane l of load i of a wavefront brings a 16-byte piece of row (4 i + wave) RPI + l / (64 / RPI); its place in the row is
  // swapped with its neighbours' by the row (xor), so that eight rows' operand reads meet every bank once.
  constexpr int LPR = 64 / Cfg::RPI;  // lanes (16-byte pieces) of a row
  const uint8_t* act_src[Cfg::LOADS];
  const int act_k = ((lane % LPR) ^ ((wave * Cfg::RPI + lane / LPR) & 7)) * 8;  // (the rows of a wavefront's loads are multiples of eight apart)
  static_assert(4 * Cfg::RPI % 8 == 0, "the same place in every load's rows");
#pragma unroll
  for (int i = 0; i < Cfg::LOADS; ++i) {
    const int r = (4 * i + wave) * Cfg::RPI + lane / LPR, pair = mine[r < rows ? r : rows - 1];
    act_src[i] = (const uint8_t*)((const T*)a.X + (int64_t)(UP ? pair / a.top_k : pair) * a.K + act_k);
  }
  const int s_begin = chunk * a.chunk_steps, s_end = s_begin + a.chunk_steps < all_steps ? s_begin + a.chunk_steps : all_steps;
  auto load_act = [&](int s) __attribute__((always_inline)) {
    const int k = s * (KSB * 128);
    const uint32_t buf = lds0 + (uint32_t)((s & 1) * Cfg::ACT);
#pragma unroll
    for (int i = 0; i < Cfg::LOADS; ++i) {
      if ((4 * i + wave) * Cfg::RPI >= rows) break;  // (uniform)
      const uint32_t at = (uint32_t)((4 * i + wave) * 1024);
      if (k + act_k < a.K) direct16(act_src[i] + k * 2, buf + at);
      else *(uint4_t*)(smem + (s & 1) * Cfg::ACT + at + lane * 16) = uint4_t{0, 0, 0, 0};
    }
  };
  // weights
  auto weight_row = [&](int t, int r) __attribute__((always_inline)) -> int64_t {
    t = tile0 + t < n_tiles ? tile0 + t : n_tiles - 1;
    return UP ? (int64_t)e * 2 * a.N + (r >> 3) * a.N + t * 8 + (r & 7) : (int64_t)e * a.N + t * 16 + r;
  };
  const uint8_t* const w_base = uniform_ptr(a.Wp + (int64_t)e * (UP ? 2 : 1) * a.N * (a.K / 2));
  uint32_t w_off[NT];  // (an expert's matrix is below 4 GiB)
#pragma unroll
  for (int t = 0; t < NT; ++t) w_off[t] = (uint32_t)((weight_row(wave * NT + t, r16) - (int64_t)e * (UP ? 2 : 1) * a.N) * (a.K / 2)) + q * 16;
  const int w_last = a.K / 2 - 16 - q * 16;
  // (global, not flat: a flat load counts as an LDS access too, and the operand reads would wait for it)
  typedef __attribute__((address_space(1))) const uint4_t* global16_t;
  uint4_t next[KSB][NT];
  auto load_weights = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < KSB; ++b) {
      const int at = (s * KSB + b) * 64;
      const uint32_t off = (uint32_t)(at < w_last ? at : w_last);
#pragma unroll
      for (int t = 0; t < NT; ++t) next[b][t] = *(global16_t)(uintptr_t)(w_base + (w_off[t] + off));
    }
  };
  // scales of window v: pieces (row * groups) / 8 + v and the next one of every row (the tensors' sizes are multiples of 16 bytes, so that
  // no piece reaches past their ends)
  const int window = a.window;
  const int64_t sc_e = (int64_t)e * (UP ? 2 : 1) * a.N * a.groups;  // the expert's first value: a multiple of eight
  const uint32_t sc_last = (uint32_t)((UP ? 2 : 1) * a.N * a.groups / 8 - 1) * 16;
  constexpr int SC_LOADS = Cfg::TILES * 32 / 256;  // (with two pieces)
  uint32_t sc_off[SC_LOADS];
#pragma unroll
  for (int i = 0; i < SC_LOADS; ++i) {
    const int c = (i * 4 + wave) * 64 + lane, r = c >> (pieces - 1);
    sc_off[i] = (uint32_t)((weight_row(r >> 4, r & 15) * a.groups - sc_e) / 8 + (pieces == 2 ? c & 1 : 0)) * 16;
  }
  const uint8_t* const sc_base = uniform_ptr((const uint8_t*)((const T*)a.scales + (a.scales ? sc_e : 0)));
  const uint8_t* const zp_base = uniform_ptr((const uint8_t*)((const T*)a.zeros + (a.zeros ? sc_e : 0)));
  auto load_scales = [&](int v) __attribute__((always_inline)) {
    const uint32_t buf = lds0 + 2 * Cfg::ACT + (uint32_t)((v & 1) * window_bytes);
#pragma unroll
    for (int i = 0; i < SC_LOADS; ++i) {
      if ((i * 4 + wave) * 1024 >= window_bytes) break;  // (uniform)
      uint32_t off = sc_off[i] + (uint32_t)v * 16;
      off = off < sc_last ? off : sc_last;
      if (a.scales) direct16_at(off, sc_base, buf + (i * 4 + wave) * 1024);
      if (ANY && a.zeros) direct16_at(off, zp_base, buf + 2 * window_bytes + (i * 4 + wave) * 1024);
    }
  };
  int sc_at[NT];  // where this lane's first scale of a window lies in it (in values); the first of window v is group 8 v
#pragma unroll
  for (int t = 0; t < NT; ++t) sc_at[t] = ((wave * NT + t) * 16 + r16) * 8 * pieces + (int)((weight_row(wave * NT + t, r16) * a.groups) & 7);
  const T one = from_float<T>(1.0f), zs = from_float<T>(a.zero_scalar);
  const NibbleMagic mg = make_nibble_magic();
  const int u_last = a.K / 32 - 1;

  auto run = [&](auto mt_tag) __attribute__((always_inline)) {
    constexpr int MT = decltype(mt_tag)::value;
    float4_t acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[t][m] = float4_t{0, 0, 0, 0};
    int v = s_begin / window, in_window = s_begin - v * window;
    for (int s = s_begin; s < s_end; ++s) {
      uint4_t w[KSB][NT];
#pragma unroll
      for (int b = 0; b < KSB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          w[b][t] = next[b][t];
          asm volatile("" : "+v"(w[b][t].x), "+v"(w[b][t].y), "+v"(w[b][t].z), "+v"(w[b][t].w));
        }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // this step's rows are there, and nobody reads the last step's any more
      if (s + 1 < s_end) {
        load_act(s + 1);
        if ((in_window == 0 || s == s_begin) && (v + 1) * window < s_end) load_scales(v + 1);
        load_weights(s + 1);
      }
      const uint8_t* const x0 = smem + (s & 1) * Cfg::ACT + r16 * Cfg::ROW_BYTES;
      const int buf = (v & 1) * (window_bytes / 2);
#pragma unroll
      for (int b = 0; b < KSB; ++b) {
        const int u = (s * KSB + b) * 4 + q, g = a.group_of(u < u_last ? u : u_last) - 8 * v + buf;
        T sv[NT], zv[NT];
        bool whole = true;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          sv[t] = a.scales ? ((const T*)sc)[sc_at[t] + g] : one;
          zv[t] = ANY && a.zeros ? ((const T*)zp)[sc_at[t] + g] : zs;
          if (ANY && kFolds<T>) whole = whole && zero_folds(to_float(zv[t]));
        }
        if ((s * KSB + b) * 128 + 128 > a.K) {  // (uniform) behind K: zeros, not an infinite weight times zero
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sv[t] = u > u_last ? from_float<T>(0.0f) : sv[t];
            zv[t] = u > u_last ? from_float<T>(0.0f) : zv[t];
          }
        }
        auto multiply = [&](auto fold_tag) __attribute__((always_inline)) {
          typedef Expand8<T, decltype(fold_tag)::value> Ex;
          Ex ex[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) ex[t] = Ex(sv[t], zv[t], mg);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            uint4_t x[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m] = *(const uint4_t*)(x0 + m * 16 * Cfg::ROW_BYTES + (((b * 16 + 4 * q + j) ^ (r16 & 7)) * 16));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const uint32_t word = j == 0 ? w[b][t].x : j == 1 ? w[b][t].y : j == 2 ? w[b][t].z : w[b][t].w;
              if constexpr (kFolds<T> && !decltype(fold_tag)::value) __builtin_amdgcn_sched_barrier(0);  // (few registers rather than fast)
              const uint4_t wo = ex[t](word);
#pragma unroll
              for (int m = 0; m < MT; ++m) acc[t][m] = Mma::mma(wo, x[m], acc[t][m]);
            }
          }
        };
        if constexpr (!kFolds<T>) {
          multiply(std::false_type{});
        } else if constexpr (ANY) {
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(whole) == ~0ull, 1)) multiply(std::true_type{});
          else multiply(std::false_type{});
        } else {
          multiply(std::true_type{});
        }
      }
      if (++in_window == window) in_window = 0, ++v;
    }
    int pair[MT];
    float weight[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      pair[m] = mine[m * 16 + r16 < rows ? m * 16 + r16 : rows - 1];
      weight[m] = UP ? 0.0f : a.weights[pair[m]];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = (tile0 + wave * NT + t) * OUTS + q * 4;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (UP && chunks > 1) {  // this lane's four gates (q = 0, 1) or ups
          if (m * 16 + r16 < rows && tile0 + wave * NT + t < n_tiles)
            *(float4_t*)((float*)a.out + ((int64_t)chunk * a.pairs + pair[m]) * (2 * (int64_t)a.N) + (q >= 2 ? a.N - 8 : 0) + n) = acc[t][m];
          continue;
        }
        moe_store<T, UP>(a, acc[t][m], m * 16 + r16 < rows && tile0 + wave * NT + t < n_tiles, pair[m], weight[m], n, q, chunk);
      }
    }
  };
  load_scales(s_begin / window);
  load_act(s_begin);
  load_weights(s_begin);
  if (rows > Cfg::ROWS / 2) run(std::integral_constant<int, MAXMT>{});
  else run(std::integral_constant<int, MAXMT / 2>{});
}

// ---- few pairs: every weight read once ---------------------------------------------------------------------------------------
// For calls that are bound by reading the weights.  A work-group stages up to `row_cap` of its expert's activation rows in LDS, whole, with
// the scales and zero points of its tiles, once; then every wavefront streams the packed weights of its own tiles through its registers,
// with no barrier: the next kFewGroup blocks (1 KB each) are on their way while the last ones are expanded and multiplied with all rows.
// No launch sorts the pairs first: a work-group looks its expert's pairs up among all ids (at most kFewPairs).  The work-groups of
// an expert are those of the first pair that names it, or, where there are more pairs than experts, those of the expert's number; one
// token's pairs are taken one by one.
//   A tile is 16 weight rows: 16 outputs, or 8 gate rows and the 8 up rows that go with them.  A block is 128 values of K of a tile.
// Where tiles are few, `splits` wavefronts share one, each with a part of K; their sums meet in LDS and are added in the order of K.
// Long rows of the down product are cut into `chunks` work-groups too, whose sums moe_combine_kernel adds.
//   fp16, zero points: one token, 6 of 64 experts of 1408 x 2048, gate / up 10.3 us (18 MB), down 9.3; 2 of 8 of 4096 x 14336, down 22 us + 4 for the sums
// (66 MB, 13.4 us at the rate of a large copy).  What is left is latency: ids, then rows and scales, then the weights of a wavefront, 4 KB at a time: 8 KB in the
// first case, 28 KB in the last.  With eight blocks asked for at once the kernel spills and takes 25 - 40 % more.
constexpr int kFewPairs = 2048;
constexpr int kFewGroup = 4;
enum { kFewByPair = 1, kFewOneToken = 2 };

struct FewArgs {
  const void* X;
  const uint8_t* Wp;
  const void* scales;
  const void* zeros;
  const float* weights;
  const int32_t* ids;
  void* out;
  int pairs, E, top_k, N, K, groups;
  uint32_t per_group;    // ceil(2^32 / (group / 32)), 0 for groups of 32 (rows of at most 65536 values: exact)
  float zero_scalar;
  int n_groups, units;   // work-groups of an expert side by side, and of all experts
  uint32_t blocks;       // blocks of 128 values of K of a work-group | 16-byte pieces of a row's scales << 16
  uint32_t shape;        // wavefronts | splits << 8 | row_cap << 16 | flags << 24
  int per_wave;          // tiles of a wavefront
};

// Where what lies in LDS, for the kernel and for the launch: activation rows, sums of the other wavefronts, scales, zero points (with a tensor of them; one
// that is a number takes no room, whole or not), the rows' weights (down), two words (number of pairs, an earlier pair has this expert), the pairs.
struct FewLds {
  int sums, scales, zeros, weights, head, list;
};
__host__ __device__ inline FewLds few_lds(bool up, bool zeros, int waves, int splits, int wg_tiles, int row_cap, int pitch, int pieces) {
  FewLds l;
  l.sums = row_cap * pitch;
  l.scales = l.sums + waves / splits * (splits - 1) * 1024;
  l.zeros = l.scales + wg_tiles * 256 * pieces;
  l.weights = l.zeros + (zeros ? wg_tiles * 256 * pieces : 0);
  l.head = l.weights + (up ? 0 : 64);
  l.list = l.head + 16;
  return l;
}

template <typename T, bool UP, bool ANY>
__global__ __launch_bounds__(512, 4) void moe_few_kernel(const FewArgs a) {
  typedef typename MmaOf<T>::type Mma;
  typedef __attribute__((address_space(3))) uint8_t* lptr_t;
  extern __shared__ __align__(16) uint8_t smem[];
  const int waves = a.shape & 255, splits = (a.shape >> 8) & 255, row_cap = (a.shape >> 16) & 255, flags = a.shape >> 24;
  const int wg_blocks = a.blocks & 0xffff, pieces = a.blocks >> 16, threads = waves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
  // neighbouring numbers go to different XCDs: those eight apart are the parts of K of one unit, which share its scales
  const int chunks = ((a.K + 127) / 128 + wg_blocks - 1) / wg_blocks;
  int unit = blockIdx.x, chunk = 0;
  if (chunks > 1) {
    const int i = unit >> 3, per8 = i / chunks;
    chunk = i - per8 * chunks;
    unit = per8 * 8 + (unit & 7);
    if (unit >= a.units) return;
  }
  const int who = unit / a.n_groups, group_no = unit - who * a.n_groups;
  const bool by_pair = flags & kFewByPair, one_token = flags & kFewOneToken;
  const int k0 = chunk * wg_blocks * 128, k_len = a.K - k0 < wg_blocks * 128 ? a.K - k0 : wg_blocks * 128;  // this work-group's part of K
  const int pitch = wg_blocks * 256 + 16;  // bytes of an activation row: 16 more, so that the rows of an operand lie on different banks
  constexpr int OUTS = UP ? 8 : 16;        // outputs of a tile
  const int wg_tiles = waves / splits * a.per_wave, n_tiles = a.N / OUTS, tile0 = group_no * wg_tiles;
  const FewLds at_lds = few_lds(UP, ANY && a.zeros, waves, splits, wg_tiles, row_cap, pitch, pieces);
  const int sums_at = at_lds.sums, sc_at = at_lds.scales, zp_at = at_lds.zeros, weights_at = at_lds.weights;
  uint8_t* const act = smem;
  int32_t* const head = (int32_t*)(smem + at_lds.head);  // [0] number of pairs, [1] an earlier pair has this expert
  uint16_t* const list = (uint16_t*)(smem + at_lds.list);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)smem);

  const int e = by_pair ? __builtin_amdgcn_readfirstlane(a.ids[who]) : who;
  const bool none = (uint32_t)e >= (uint32_t)a.E;
  if (none && (!UP || by_pair)) {
    if (!UP) return;
    T* const h = (T*)a.out + (int64_t)who * a.N;
    const int end = (tile0 + wg_tiles) * OUTS;
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
    const int width = wg_tiles * OUTS;
    for (int i = tid; i < count * width; i += threads) {
      const int n = tile0 * OUTS + i % width;
      if (n < a.N) h[(int64_t)list[i / width] * a.N + n] = from_float<T>(0.0f);
    }
    return;
  }

  // the row of W that row r of tile t is
  auto weight_row = [&](int t, int r) __attribute__((always_inline)) -> int64_t {
    t = t < n_tiles ? t : n_tiles - 1;
    return UP ? (int64_t)e * 2 * a.N + (r >> 3) * a.N + t * 8 + (r & 7) : (int64_t)e * a.N + t * 16 + r;
  };
  auto group_of = [&](int u) __attribute__((always_inline)) -> int {  // the group of the u-th 32 values of a row
    return a.per_group ? (int)__umulhi((uint32_t)u, a.per_group) : u;
  };
  // a pass's rows -> LDS, 1 KB an instruction; and zeros up to the end of the last block
  auto load_rows = [&](int row0, int rows) __attribute__((always_inline)) {
    const int per_row = (k_len + 511) >> 9;
    if (!UP && wave == 0 && lane < rows) direct4(a.weights + (one_token ? who : (int)list[row0 + lane]), lds0 + weights_at);
    for (int i = wave; i < rows * per_row; i += waves) {
      const int r = i / per_row, at = (i - r * per_row) * 1024;
      const int pair = one_token ? who : __builtin_amdgcn_readfirstlane((int)list[row0 + r]);
      const uint8_t* const x = (const uint8_t*)((const T*)a.X + (int64_t)(UP ? pair / a.top_k : pair) * a.K + k0);
      if (at + lane * 16 < k_len * 2) direct16(x + at + lane * 16, lds0 + r * pitch + at);
      else if (at + lane * 16 < ((k_len + 127) & ~127) * 2) *(uint4_t*)(act + r * pitch + at + lane * 16) = uint4_t{0, 0, 0, 0};
    }
  };
  // Scales and zero points of the work-group's tiles and part of K: for each of 16 rows a tile the `pieces` 16-byte pieces that hold them.
  // A row's first value lies (row * groups + g0) % 8 values into its first piece; the tensors' sizes are multiples of 16 bytes, so that
  // no piece reaches past their ends.
  const int g0 = group_of(k0 / 32);
  {
    const int all = wg_tiles * 16 * pieces;
    const int64_t end = (int64_t)a.E * (UP ? 2 : 1) * a.N * a.groups;
    // (no load into registers is on its way here; said so, because the compiler would wait for one ahead of the weights, and so for the
    // direct loads)
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    for (int c0 = wave * 64; c0 < all; c0 += threads) {
      const int c = c0 + lane;
      if (c >= all) continue;
      const int r = c / pieces, at = c - r * pieces;
      int64_t off = (weight_row(tile0 + (r >> 4), r & 15) * a.groups + g0) / 8 * 8 + at * 8;
      off = off < end ? off : end - 8;
      if (a.scales) direct16((const T*)a.scales + off, lds0 + sc_at + c0 * 16);
      if (ANY && a.zeros) direct16((const T*)a.zeros + off, lds0 + zp_at + c0 * 16);
    }
  }

  // this wavefront's part of K and tiles
  const int lane_tile = wave / splits, split = wave - lane_tile * splits, my_tile0 = lane_tile * a.per_wave;
  const int blocks = (k_len + 127) >> 7, per = (wg_blocks + splits - 1) / splits, block0 = split * per;
  const int mine = blocks - block0 < per ? (blocks - block0 < 0 ? 0 : blocks - block0) : per;
  int my_tiles = n_tiles - tile0 - my_tile0;
  my_tiles = my_tiles < 0 ? 0 : my_tiles < a.per_wave ? my_tiles : a.per_wave;
  const int total = my_tiles * mine;
  // lane (r16, q) loads the 32 values 32 q .. of each block of row r16; past the end of a row its last ones (behind K the activation rows
  // in LDS are zeros)
  const uint8_t* const w_first = a.Wp + weight_row(tile0 + my_tile0, r16) * (a.K / 2);
  const int64_t tile_stride = (int64_t)OUTS * (a.K / 2);
  const int off_first = k0 / 2 + block0 * 64 + q * 16, off_last = a.K / 2 - 16;
  const T one = from_float<T>(1.0f), zs = from_float<T>(a.zero_scalar);
  const NibbleMagic mg = make_nibble_magic();
  const int u_last = a.K / 32 - 1;

  for (int row0 = 0; row0 < count; row0 += row_cap) {
    const int rows = count - row0 < row_cap ? count - row0 : row_cap;
    if (row0) __syncthreads();  // (the last pass's rows have been read, its sums added up)
    load_rows(row0, rows);
    // the first group, and how to go on from there: loads into registers behind the direct ones
    uint4_t next[kFewGroup];
    const uint8_t* src = w_first;
    int load_block = 0, load_tile = 0;
    auto load_group = [&]() __attribute__((always_inline)) {  // always kFewGroup loads, past the last tile of its last block
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        const int off = off_first + load_block * 64;
        next[i] = __builtin_nontemporal_load((const uint4_t*)(src + (off < off_last ? off : off_last)));
        if (load_block + 1 < mine) ++load_block;
        else if (load_tile + 1 < my_tiles) load_block = 0, ++load_tile, src += tile_stride;
      }
    };
    // wait for the rows and, ahead of the first pass, the scales
    if (total > 0) {
      load_group();
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kFewGroup) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();

    const int my_row = r16 < rows ? r16 : rows - 1, my_pair = list[row0 + my_row];
    const float my_weight = UP ? 0.0f : *(const float*)(smem + weights_at + my_row * 4);
    const uint8_t* const my_act = act + my_row * pitch + q * 64 + block0 * 256;
    float4_t acc[2] = {float4_t{0, 0, 0, 0}, float4_t{0, 0, 0, 0}};
    int tile = 0, block = 0, sc0 = 0;
    for (int s = 0; s < total; s += kFewGroup) {
      uint4_t w[kFewGroup];
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        w[i] = next[i];
        asm volatile("" : "+v"(w[i].x), "+v"(w[i].y), "+v"(w[i].z), "+v"(w[i].w));
      }
      if (s + kFewGroup < total) load_group();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        if (s + i >= total) break;
        if (block == 0)  // this lane's scales in LDS: that of group g lies at sc0 + g
          sc0 = ((my_tile0 + tile) * 16 + r16) * pieces * 8 + (int)((weight_row(tile0 + my_tile0 + tile, r16) * a.groups + g0) & 7) - g0;
        const int u = k0 / 32 + (block0 + block) * 4 + q, at = sc0 + group_of(u < u_last ? u : u_last);
        T sv = a.scales ? ((const T*)(smem + sc_at))[at] : one, zv = ANY && a.zeros ? ((const T*)(smem + zp_at))[at] : zs;
        if (u > u_last) sv = zv = from_float<T>(0.0f);  // (behind K: zeros, not an infinite weight times zero)
        const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        const uint8_t* const x = my_act + block * 256;
        auto multiply = [&](auto fold_tag) __attribute__((always_inline)) {
          const Expand8<T, decltype(fold_tag)::value> ex(sv, zv, mg);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j & 1] = Mma::mma(ex(words[j]), *(const uint4_t*)(x + j * 16), acc[j & 1]);
        };
        if constexpr (!kFolds<T>) {
          multiply(std::false_type{});
        } else if constexpr (ANY) {
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(zero_folds(to_float(zv))) == ~0ull, 1)) multiply(std::true_type{});
          else multiply(std::false_type{});
        } else {
          multiply(std::true_type{});
        }
        if (++block < mine) continue;
        block = 0;
        if (splits == 1) {
          moe_store<T, UP>(a, acc[0] + acc[1], r16 < rows, my_pair, my_weight, (tile0 + my_tile0 + tile) * OUTS + q * 4, q, chunk);
          acc[0] = acc[1] = float4_t{0, 0, 0, 0};
        }
        ++tile;
      }
    }
    if (splits > 1) {  // (one tile a wavefront) the sums of the others
      float4_t sum = acc[0] + acc[1];
      float* const sums = (float*)(smem + sums_at) + (lane_tile * (splits - 1) * 64 + lane) * 4;
      if (split) *(float4_t*)(sums + (split - 1) * 256) = sum;
      __syncthreads();
      if (split == 0 && my_tiles > 0) {
        for (int i = 1; i < splits; ++i) sum += *(const float4_t*)(sums + (i - 1) * 256);
        moe_store<T, UP>(a, sum, r16 < rows, my_pair, my_weight, (tile0 + my_tile0) * OUTS + q * 4, q, chunk);
      }
    }
  }
}

// (down of 4099 tokens, 6 slots of 2048: 32 us for 218 MB, 6.9 TB/s.)  y[t] = the sum of token t's rows, slot by slot, each over the parts of K it was cut into; four slots' rows are asked for at once.  A
// work-group has 256 x 4 values of one token.
__global__ __launch_bounds__(256) void moe_combine_kernel(const float* __restrict__ rows, const int32_t* __restrict__ ids, void* __restrict__ Y,
                                                         int N, int n_groups, int top_k, int E, int out_dtype, int chunks, int64_t chunk_stride) {
  const int64_t t = blockIdx.x / (uint32_t)n_groups;
  const int n = ((int)(blockIdx.x - (uint32_t)t * n_groups) * 256 + (int)threadIdx.x) * 4;
  if (n >= N) return;
  const int32_t* const my_ids = ids + t * top_k;
  const float* const mine = rows + t * top_k * N + n;
  float4_t sum{0, 0, 0, 0};
  for (int j = 0; j < top_k; j += 4) {
    float4_t v[4];
    bool there[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      there[i] = j + i < top_k && (uint32_t)my_ids[j + i] < (uint32_t)E;  // (otherwise no row was written)
      v[i] = there[i] ? *(const float4_t*)(mine + (int64_t)(j + i) * N) : float4_t{0, 0, 0, 0};
    }
    for (int c = 1; c < chunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (there[i]) v[i] += *(const float4_t*)(mine + c * chunk_stride + (int64_t)(j + i) * N);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (there[i]) sum += v[i];
  }
  const int64_t o = t * N + n;
  if (out_dtype == TLQ_F32) {
    *(float4_t*)((float*)Y + o) = sum;
  } else if (out_dtype == TLQ_F16) {
    const half_t h[4] = {(half_t)sum[0], (half_t)sum[1], (half_t)sum[2], (half_t)sum[3]};
    *(uint2_t*)((half_t*)Y + o) = bitcast<uint2_t>(h);
  } else {
    *(uint2_t*)((uint16_t*)Y + o) = uint2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

// h of the gate / up product from its sums over parts of K.  A work-group has 256 x 4 values of one pair.
template <typename T>
__global__ __launch_bounds__(256) void moe_gate_kernel(const float* __restrict__ parts, const int32_t* __restrict__ ids, T* __restrict__ H, int N,
                                                      int n_groups, int E, int chunks, int64_t chunk_stride) {
  const int64_t pair = blockIdx.x / (uint32_t)n_groups;
  const int n = ((int)(blockIdx.x - (uint32_t)pair * n_groups) * 256 + (int)threadIdx.x) * 4;
  if (n >= N) return;
  T o[4];
  if ((uint32_t)ids[pair] < (uint32_t)E) {
    const float* const mine = parts + pair * 2 * N + n;
    float4_t g = *(const float4_t*)mine, u = *(const float4_t*)(mine + N);
    for (int c = 1; c < chunks; ++c) g += *(const float4_t*)(mine + c * chunk_stride), u += *(const float4_t*)(mine + c * chunk_stride + N);
    const float4_t y = silu_times(g, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = from_float<T>(y[i]);
  } else {  // (no row was written)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = from_float<T>(0.0f);
  }
  *(uint2_t*)(H + pair * N + n) = bitcast<uint2_t>(o);
}

int check_experts(const char* what, int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K, int64_t group, int dtype) {
  TLQ_REQUIRE(M >= 0 && M < ((int64_t)1 << 32) && E >= 1 && E <= kMaxExperts && top_k >= 1 && top_k <= 64, "%s: bad shape M=%lld E=%lld top_k=%lld (at most 1024 experts, 64 of them for a token)",
              what, (long long)M, (long long)E, (long long)top_k);
  TLQ_REQUIRE(M * top_k < ((int64_t)1 << 24), "%s: M * top_k = %lld is 2^24 or more: call it for fewer tokens at once", what, (long long)(M * top_k));
  TLQ_REQUIRE(N >= 16 && N % 16 == 0 && N < ((int64_t)1 << 24), "%s: N=%lld must be a multiple of 16", what, (long long)N);
  TLQ_REQUIRE(K >= 32 && K % 32 == 0 && K < ((int64_t)1 << 24), "%s: K=%lld must be a multiple of 32", what, (long long)K);
  TLQ_REQUIRE(group >= 32 && group % 32 == 0 && K % group == 0, "%s: group=%lld must be a multiple of 32 that divides K=%lld", what,
              (long long)group, (long long)K);
  TLQ_REQUIRE(2 * N * (K / 2) < ((int64_t)1 << 32), "%s: N=%lld x K=%lld is too large a matrix for one expert", what, (long long)N, (long long)K);
  TLQ_REQUIRE(dtype == TLQ_F16 || dtype == TLQ_BF16, "%s: in_dtype must be float16 or bfloat16 (got %d)", what, dtype);
  return 0;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// How moe_few_kernel is launched.  ok: it takes the call.
struct FewPlan {
  bool ok;
  int waves, splits, per_wave, row_cap, n_groups, chunks, blocks, pieces;
  bool by_pair;
  int64_t lds, units, grid;
};
int64_t few_chunks(int64_t K) { return ceil_div(ceil_div(K, (int64_t)128), (int64_t)32); }
FewPlan few_plan(bool up, int64_t pairs, int64_t E, int64_t top_k, int64_t N, int64_t K, int64_t group, bool zeros) {
  FewPlan p{};
  const int64_t all = ceil_div(K, (int64_t)128), n_tiles = N / (up ? 8 : 16);
  const int64_t experts = pairs < E ? pairs : E;
  if (pairs > kFewPairs || K > 65536) return p;
  p.chunks = up ? 1 : (int)few_chunks(K);
  const int64_t blocks = ceil_div(all, (int64_t)p.chunks);
  p.chunks = (int)ceil_div(all, blocks);
  p.blocks = (int)blocks;
  p.waves = 4;
  p.splits = 1;
  while (p.splits < 4 && p.splits * 4 <= blocks && experts * n_tiles * p.chunks * p.splits < 2048) p.splits *= 2;
  p.per_wave = 1;
  // tiles of a wavefront: as many as leave every CU several work-groups (gate / up is on tiles of pairs where there are that many, few_pairs)
  if (!up && p.splits == 1)
    while (p.per_wave < 8 && experts * ceil_div(n_tiles, (int64_t)p.waves * p.per_wave * 2) * p.chunks >= 1536) p.per_wave *= 2;
  p.by_pair = pairs <= E;
  // the scales of a part of K: its groups, the first of them anywhere in its piece; parts need not begin with a group
  const int64_t part_groups = p.chunks == 1 ? K / group : (blocks * 128 + group - 1) / group + 1;
  p.pieces = (int)((part_groups + 7 + 7) / 8);
  // rows of a pass: sixteen (an operand's columns), while they leave LDS for two work-groups
  const int64_t pitch = blocks * 256 + 16;
  p.row_cap = 16;
  while (p.row_cap > 1 && (p.row_cap > pairs || p.row_cap * pitch > 36 * 1024)) p.row_cap /= 2;
  if (p.by_pair && pairs == top_k) p.row_cap = 1;
  const int64_t wg_tiles = p.waves / p.splits * p.per_wave;
  p.n_groups = (int)ceil_div(n_tiles, wg_tiles);
  p.lds = few_lds(up, zeros, p.waves, p.splits, (int)wg_tiles, p.row_cap, (int)pitch, p.pieces).list + ceil_div(pairs, (int64_t)8) * 16;
  p.units = (p.by_pair ? pairs : E + (up ? 1 : 0)) * p.n_groups;
  p.grid = p.chunks == 1 ? p.units : ceil_div(p.units, (int64_t)8) * 8 * p.chunks;
  p.ok = p.lds <= 160 * 1024 && p.grid <= kMostGroups;
  return p;
}

template <typename T, bool UP, bool ZEROS>
int launch_few(const char* what, const FewArgs& a, const FewPlan& p, hipStream_t st) {
  auto kern = moe_few_kernel<T, UP, ZEROS>;
  static bool attr_set = false;
  if (!attr_set) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    TLQ_REQUIRE(e == hipSuccess, "%s: cannot reserve LDS: %s", what, hipGetErrorString(e));
    attr_set = true;
  }
  kern<<<(unsigned)p.grid, p.waves * 64, (size_t)p.lds, st>>>(a);
  return check_launch(what, "moe_few_kernel") ? 0 : 1;
}

template <bool UP>
int run_few(const char* what, const ExpertArgs& x, const void* ids, int64_t pairs, int dtype, const FewPlan& p, hipStream_t st) {
  const bool whole = zero_folds(x.zero_scalar);
  const int units = x.group / 32;
  const int flags = (p.by_pair ? kFewByPair : 0) | (p.by_pair && pairs == x.top_k ? kFewOneToken : 0);
  const FewArgs a{x.X, x.Wp, x.scales, x.zeros, x.weights, (const int32_t*)ids, x.out, (int)pairs, x.E, x.top_k, x.N, x.K, x.K / x.group,
                  units == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + units - 1) / units), x.zero_scalar, p.n_groups, (int)p.units,
                  (uint32_t)(p.blocks | p.pieces << 16), (uint32_t)(p.waves | p.splits << 8 | p.row_cap << 16 | flags << 24), p.per_wave};
#define TLQ_FEW(T) (x.zeros || !whole ? launch_few<T, UP, true>(what, a, p, st) : launch_few<T, UP, false>(what, a, p, st))
  return dtype == TLQ_F16 ? TLQ_FEW(half_t) : TLQ_FEW(bf16_t);
#undef TLQ_FEW
}

template <typename T, bool UP, bool ZEROS, int MAXMT, int NT, int KSB>
int launch_tiles(const char* what, const TileArgs& a, int64_t grid, hipStream_t st) {
  auto kern = moe_tile_kernel<T, UP, ZEROS, MAXMT, NT, KSB>;
  const int lds = TileCfg<MAXMT, NT, KSB>::lds(a.groups % 8 == 0 ? 1 : 2, a.zeros != nullptr);
  static bool attr_set = false;
  if (!attr_set) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, TileCfg<MAXMT, NT, KSB>::lds(2, true));
    TLQ_REQUIRE(e == hipSuccess, "%s: cannot reserve LDS: %s", what, hipGetErrorString(e));
    attr_set = true;
  }
  kern<<<(unsigned)grid, 256, (size_t)lds, st>>>(a);
  return check_launch(what, "moe_tile_kernel") ? 0 : 1;
}

// Work-groups of moe_tile_kernel side by side, and the parts that K is cut into where there are too few of them
// to keep four on every CU (down of eight experts of 4096 x 14336 and 16 tokens: 106 us whole).  `tiles`: about how many tiles of pairs there are.
template <bool UP, int NT>
int64_t tile_groups(int64_t N) {
  return ceil_div(N, (int64_t)(4 * NT * (UP ? 8 : 16)));
}
int64_t tile_chunks(int64_t tiles, int64_t n_groups, int64_t K) {
  int64_t chunks = 1;
  while (chunks < 8 && tiles * n_groups * chunks * 2 <= 1024 && K / (chunks * 2) >= 1024) chunks *= 2;
  return chunks;
}
int64_t about_tiles(int64_t pairs, int64_t E, int64_t rows) { return (pairs < E ? pairs : E) + pairs / rows; }

// The plan, then the products on tiles of 16 MAXMT pairs.  chunks: the parts of K.
template <bool UP, int MAXMT, int NT, int KSB>
int run_tiles(const char* what, const ExpertArgs& x, const void* ids, int64_t pairs, int dtype, void* ws, int64_t* chunks, hipStream_t st, bool large = false) {
  constexpr int rows = 16 * MAXMT;
  static_assert(rows == 32 || rows == 64, "sizes that the workspace holds the plan of");
  const PlanSizes z = plan_sizes(x.E, pairs, rows, large);
  const PlanPtrs p = plan_at(ws, pairs, z);
  const int64_t n_groups = tile_groups<UP, NT>(x.N), steps = ceil_div((int64_t)x.K, (int64_t)(KSB * 128));
  const int64_t chunk_steps = large ? steps : ceil_div(steps, tile_chunks(about_tiles(pairs, x.E, rows), n_groups, x.K));
  *chunks = ceil_div(steps, chunk_steps);
  float* const parts = UP && *chunks > 1 ? (float*)((uint8_t*)ws + plan_bytes(x.E, pairs)) : nullptr;
  const int64_t grid = z.small * n_groups * *chunks;
  TLQ_REQUIRE(grid <= kMostGroups, "%s: %lld work-groups: call it for fewer tokens at once", what, (long long)grid);
#define TLQ_PLAN(COMPACT, THREADS)                                                                                                          \
  moe_plan_kernel<COMPACT, THREADS><<<x.E + 1, THREADS, 0, st>>>((const int32_t*)ids, p.totals, p.order, p.small, p.large, (int)pairs, x.E, rows, \
                                                                 large ? (int)moe_panel_groups(x.N, UP) : 0)
  if (pairs > kCompactPairs) TLQ_PLAN(false, kPlanThreads);
  else if (pairs > kCompactPairs / 4) TLQ_PLAN(true, kPlanThreads);
  else TLQ_PLAN(true, kPlanThreads / 4);
#undef TLQ_PLAN
  if (!check_launch(what, "moe_plan_kernel")) return 1;
  if (z.large > 0) {
    const Plan plan{p.order, p.small, p.large, p.totals};
    if (moe_panel(what, x, plan, z.large, dtype, UP, st)) return 1;
  }
  const bool whole = zero_folds(x.zero_scalar);
  const int units = x.group / 32, window = units * 2 / KSB;  // steps of eight groups
  const TileArgs a{x.X, x.Wp, x.scales, x.zeros, x.weights, parts ? (void*)parts : x.out, p.small, p.order, (int)pairs, x.E, x.top_k, x.N, x.K, x.K / x.group,
                   make_group_of(units), x.zero_scalar, (int)n_groups, window, (int)chunk_steps};
#define TLQ_TILES(T) (x.zeros || !whole ? launch_tiles<T, UP, true, MAXMT, NT, KSB>(what, a, grid, st) : launch_tiles<T, UP, false, MAXMT, NT, KSB>(what, a, grid, st))
  if (dtype == TLQ_F16 ? TLQ_TILES(half_t) : TLQ_TILES(bf16_t)) return 1;
#undef TLQ_TILES
  if (!parts) return 0;
  const int64_t groups = ceil_div((int64_t)x.N, (int64_t)1024), stride = pairs * 2 * x.N;  // (few work-groups: K was cut because tiles are few)
  const dim3 g((unsigned)(pairs * groups));
  if (dtype == TLQ_F16)
    moe_gate_kernel<half_t><<<g, 256, 0, st>>>(parts, (const int32_t*)ids, (half_t*)x.out, x.N, (int)groups, x.E, (int)*chunks, stride);
  else
    moe_gate_kernel<bf16_t><<<g, 256, 0, st>>>(parts, (const int32_t*)ids, (bf16_t*)x.out, x.N, (int)groups, x.E, (int)*chunks, stride);
  return check_launch(what, "moe_gate_kernel") ? 0 : 1;
}

// Which kernel: the one without a plan while an expert has two pairs at most on average and the tiles' work-groups would not fill the machine
// (MoE layers of 8 to 256 experts, bf16, group 128, zero points, this kernel / tiles of 32: 4 tokens on 6 of 64 experts of 1408 x 2048 21.3 / 24.2 us, 8 tokens
// 30.3 / 30.0; 1 token on 2 of 8 experts, down, 4096 x 14336 25.6 / 95.8; 16 tokens on 4 of 16 experts of 2048 x 2048 28.3 / 24.5).
//   And while the passes of its `row_cap` rows stay few, each of which reads the expert's weights again: up to twice as many tokens, or pairs on few of
// the experts (groups of 32; gate / up of 256 experts of 320 x 6016, two rows a pass, 16 tokens on 2 each 30 / 54, 32 tokens 126 / 56; down of 32 of
// 640 x 10240, four rows, 4 tokens on 4 each 23 / 30, 16 tokens 61 / 36).
bool few_pairs(bool up, int64_t pairs, int64_t E, int64_t N) {
  const int64_t experts = pairs < E ? pairs : E, groups = up ? tile_groups<true, 2>(N) : tile_groups<false, 2>(N);
  return pairs <= 2 * experts && experts * groups <= 1024;
}

// Tiles of 32 pairs, 64 or 256, by the pairs of an expert on average.
//   64 rather than 32 (us, bf16, zero points; 32 / 64): gate / up of 64 experts of 1408 x 2048, 12 pairs each 58.7 / 62.2, 24 75.4 / 75.1, 40 96.5 / 92.4;
// 8 of 14336 x 4096, 12 155 / 163, 24 188 / 184, 40 268 / 221; down of 8 of 4096 x 14336, 12 94 / 97, 24 117 / 105; 16 of 2048 x 4096, 24 38.3 / 41.5, 40 50.7 / 44.5.
//   256 beside 64: where the plan can count what they make (choose by rounds, above), or with long enough rows and many pairs.  (64 / 256) gate / up of
// 64 experts of 1408 x 2048, 192 pairs each 235 / 266, 256 305 / 303, 768 791 / 615; 128 of 768 x 2048, 256 325 / 318, 768 871 / 659; down of 64 of
// 2048 x 1408, 256 193 / 224, 768 514 / 525; 128 of 2048 x 768, 768 750 / 796; 16 of 2048 x 4096, 768 326 / 325; gate / up with shorter rows, 64 of
// 1984 x 1536, 300 375 / 343, 640 737 / 579; 32 of 4096 x 1024, 300 284 / 302, 640 548 / 457; 64 of 2048 x 512, 300 165 / 178, 640 320 / 296.
constexpr int kTilesOf64 = 24, kTilesOf256 = 256, kTilesOf256Short = 448;

enum { kMoeFew = 1, kMoeTiles32 = 2, kMoeTiles64 = 3, kMoeTiles256 = 4 };
int choose_kernel(bool up, const ExpertArgs& a, int64_t pairs, FewPlan* few) {
  if (few_pairs(up, pairs, a.E, a.N)) {
    *few = few_plan(up, pairs, a.E, a.top_k, a.N, a.K, a.group, a.zeros != nullptr);
    if (few->ok && (pairs <= 2 * few->row_cap * a.top_k || pairs * 16 <= (int64_t)a.E * few->row_cap)) return kMoeFew;
  }
  if (pairs / a.E < kTilesOf64) return kMoeTiles32;
  const int64_t large_groups = pairs / kLargeRows * moe_panel_groups(a.N, up);
  const bool long_rows = a.K >= (up ? 1536 : 2048), many = up && a.K >= 512 && !long_rows ? pairs / a.E >= kTilesOf256Short : long_rows && pairs / a.E >= kTilesOf256;
  return (pairs > kCompactPairs ? many && large_groups >= 512 : large_groups >= 192) && moe_panel_takes(a, pairs, up) ? kMoeTiles256 : kMoeTiles64;
}

template <bool UP>
int run_experts(const char* what, const ExpertArgs& a, const void* ids, int64_t pairs, int dtype, void* ws, int64_t* chunks, hipStream_t st) {
  FewPlan few;
  const int kernel = choose_kernel(UP, a, pairs, &few);
  if (kernel == kMoeFew) {
    *chunks = few.chunks;
    return run_few<UP>(what, a, ids, pairs, dtype, few, st);
  }
  if (kernel == kMoeTiles32) return run_tiles<UP, 2, 2, 2>(what, a, ids, pairs, dtype, ws, chunks, st);
  return run_tiles<UP, 4, 2, 1>(what, a, ids, pairs, dtype, ws, chunks, st, kernel == kMoeTiles256);
}

// The most parts of K times pairs that a product of these pairs or of fewer has sums for: fewer pairs can make more of them (tile_chunks, few_pairs), and a
// workspace for a program's largest call has to do for the others.  0: no sums of parts (gate / up alone).
template <bool UP>
int64_t most_rows(int64_t pairs, int64_t E, int64_t top_k, int64_t N, int64_t K) {
  const int64_t groups = tile_groups<UP, 2>(N);
  int64_t most = UP ? 0 : pairs;
  const auto take = [&](int64_t chunks, int64_t up_to) {
    const int64_t rows = chunks * ((up_to < pairs ? up_to : pairs) / top_k * top_k);
    most = rows > most ? rows : most;
  };
  if (!UP) take(few_chunks(K), E * groups <= 1024 ? 2 * E : 1024 / groups);
  for (int64_t chunks = 2; chunks <= 8 && K / chunks >= 1024; chunks *= 2) {
    const int64_t tiles = 1024 / (groups * chunks);  // about_tiles at most
    if (tiles == 0) break;
    for (int64_t rows = 32; rows <= 64; rows *= 2)
      take(chunks, tiles < E ? tiles - (tiles + 1) / (rows + 1) : (tiles - E + 1) * rows - 1 > E ? (tiles - E + 1) * rows - 1 : E);
  }
  return most;
}
// of the plan alone; 0: sizes that no call takes
int64_t plan_workspace(int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K) {
  if (M <= 0 || E < 1 || top_k < 1 || E > kMaxExperts || top_k > 64 || M >= ((int64_t)1 << 24) || N < 1 || N >= ((int64_t)1 << 24) || K < 1 || K >= ((int64_t)1 << 24))
    return 0;
  return plan_bytes(E, M * top_k);
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int64_t tlq_moe_gate_up_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K) {
  const int64_t plan = plan_workspace(M, E, top_k, N, K);
  return plan + (plan ? most_rows<true>(M * top_k, E, top_k, N, K) * 2 * N * 4 : 0);
}

extern "C" int64_t tlq_moe_down_workspace_bytes(int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K) {
  const int64_t plan = plan_workspace(M, E, top_k, N, K);
  return plan + (plan ? most_rows<false>(M * top_k, E, top_k, N, K) * N * 4 : 0);
}

extern "C" int tlq_moe_gate_up_w4a16(const void* X, const void* ids, const void* w_packed, const void* scales, const void* zeros, void* H,
                                     void* workspace, int64_t workspace_bytes, int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K,
                                     int64_t group, float zero_scalar, int dtype, void* stream) {
  const char* const what = "tlq_moe_gate_up_w4a16";
  if (check_experts(what, M, E, top_k, N, K, group, dtype)) return 1;
  if (M == 0) return 0;
  TLQ_REQUIRE(X && ids && w_packed && H, "%s: null pointer", what);
  TLQ_REQUIRE(aligned16(X) && aligned16(w_packed) && aligned16(H) && aligned16(scales) && aligned16(zeros) && ((uintptr_t)ids & 3) == 0,
              "%s: X, w_packed, scales, zeros and H must be 16-byte aligned, ids to their type", what);
  const int64_t want = tlq_moe_gate_up_workspace_bytes(M, E, top_k, N, K);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && aligned16(workspace), "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  ExpertArgs a{X, (const uint8_t*)w_packed, scales, zeros, nullptr, H, (int)E, (int)top_k, (int)N, (int)K, (int)group, zero_scalar};
  int64_t chunks = 1;
  return run_experts<true>(what, a, ids, M * top_k, dtype, workspace, &chunks, (hipStream_t)stream);
}

extern "C" int tlq_moe_down_w4a16(const void* H, const void* ids, const void* weights, const void* w_packed, const void* scales,
                                  const void* zeros, void* Y, void* workspace, int64_t workspace_bytes, int64_t M, int64_t E, int64_t top_k,
                                  int64_t N, int64_t K, int64_t group, float zero_scalar, int in_dtype, int out_dtype, void* stream) {
  const char* const what = "tlq_moe_down_w4a16";
  if (check_experts(what, M, E, top_k, N, K, group, in_dtype)) return 1;
  TLQ_REQUIRE(out_dtype == TLQ_F16 || out_dtype == TLQ_BF16 || out_dtype == TLQ_F32, "%s: out_dtype must be float16, bfloat16 or float32 (got %d)", what, out_dtype);
  if (M == 0) return 0;
  TLQ_REQUIRE(H && ids && weights && w_packed && Y, "%s: null pointer", what);
  TLQ_REQUIRE(aligned16(H) && aligned16(w_packed) && aligned16(Y) && aligned16(scales) && aligned16(zeros) && (((uintptr_t)ids | (uintptr_t)weights) & 3) == 0,
              "%s: H, w_packed, scales, zeros and Y must be 16-byte aligned, ids and weights to their type", what);
  const int64_t want = tlq_moe_down_workspace_bytes(M, E, top_k, N, K);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && aligned16(workspace), "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  const int64_t pairs = M * top_k;
  float* const rows = (float*)((uint8_t*)workspace + plan_bytes(E, pairs));
  ExpertArgs a{H, (const uint8_t*)w_packed, scales, zeros, (const float*)weights, rows, (int)E, (int)top_k, (int)N, (int)K, (int)group, zero_scalar};
  hipStream_t st = (hipStream_t)stream;
  int64_t chunks = 1;
  if (run_experts<false>(what, a, ids, pairs, in_dtype, workspace, &chunks, st)) return 1;
  const int64_t n_groups = ceil_div(N, (int64_t)1024);
  const int64_t most = kMostGroups / n_groups;  // tokens of a launch
  for (int64_t t = 0; t < M; t += most) {
    const int64_t tokens = M - t < most ? M - t : most;
    moe_combine_kernel<<<(unsigned)(tokens * n_groups), 256, 0, st>>>(rows + t * top_k * N, (const int32_t*)ids + t * top_k,
                                                                      (uint8_t*)Y + t * N * (out_dtype == TLQ_F32 ? 4 : 2), (int)N, (int)n_groups, (int)top_k,
                                                                      (int)E, out_dtype, (int)chunks, pairs * N);
    if (!check_launch(what, "moe_combine_kernel")) return 1;
  }
  return 0;
}

extern "C" int tlq_debug_moe_choice(int up, int64_t M, int64_t E, int64_t top_k, int64_t N, int64_t K, int64_t group, int zeros, void* plan_out) {
  if (check_experts("tlq_debug_moe_choice", M, E, top_k, N, K, group, TLQ_F16) || M == 0) return 0;
  const ExpertArgs a{nullptr, nullptr, nullptr, zeros ? (const void*)16 : nullptr, nullptr, nullptr, (int)E, (int)top_k, (int)N, (int)K, (int)group, 0.0f};
  FewPlan few;
  const int kernel = choose_kernel(up != 0, a, M * top_k, &few);
  if (plan_out && kernel == kMoeFew) {
    const int wg_tiles = few.waves / few.splits * few.per_wave;
    const FewLds l = few_lds(up != 0, zeros != 0, few.waves, few.splits, wg_tiles, few.row_cap, few.blocks * 256 + 16, few.pieces);
    const int64_t plan[7] = {few.row_cap, few.splits, few.per_wave, few.chunks, few.lds, l.list + M * top_k * 2, few.n_groups};
    for (int i = 0; i < 7; ++i) ((int64_t*)plan_out)[i] = plan[i];
  }
  return kernel;
}

extern "C" int64_t tlq_debug_moe_group(int64_t group, int64_t u) {
  if (group < 32 || group % 32 != 0 || group >= ((int64_t)1 << 24) || u < 0 || u >= ((int64_t)1 << 19)) return -1;
  return make_group_of((int)(group / 32))((int)u);
}
