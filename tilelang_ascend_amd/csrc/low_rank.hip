// Low-rank adapters of many requests beside a projection of up to three parts side by side (queries, keys, values; gate and up):
//   out[m, n] = rn(Y[m, n] + scaling[l] * sum_j h[m, p r + j] * B[l, n, j]),  h[m, i] = sum_k X[m, k] * A[l, i, k]
// l = ids[m], p the part that n lies in, r the rank; a row whose id names no adapter is out = Y.  h and the sums are fp32, rounded once, at the end.
//
// Memory bound: Y and out, X, and the weights of the adapters that some row names, each once.  Few rows of low rank take one launch, a work-group a row and run of
// outputs.  More are gathered by adapter into tiles of 16 or 64, which meet their adapter's weights on the matrix units: the first product writes fp32 sums of
// parts of K (few tiles: many parts), the second adds the parts as it reads them.  A row's values do not depend on its tile or its place there.
#include "gemm_core.h"

namespace tlq {
namespace {

constexpr int kInlineRows = 64;  // up to here a wavefront looks at all ids itself and no plan is made
constexpr int kMaxAdapters = 4096;

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

// Global -> LDS without registers: 16 bytes a lane, lane l's to lds + 16 l.  (Between the write of M0 and the load that reads it
// the hardware wants a wait state, which the compiler inserts behind its builtins alone: s_nop.)
__device__ __forceinline__ void direct16(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(lds), "v"(src) : "memory");
}
typedef __attribute__((address_space(3))) uint8_t* lptr_t;
__device__ __forceinline__ uint32_t lds_of(const void* p) { return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)p); }

// ---- which rows ---------------------------------------------------------------------------------------------------------
// A tile: `rows` rows of one adapter (L: rows without one), those of the plan's order from `first` on.
struct RowTile {
  int32_t adapter, first, rows, unused;
};
// plan: [0] how many tiles there are; from 64 on the rows by adapter, then the tiles.
struct Rows {
  const int32_t *ids, *plan;  // plan: null up to kInlineRows rows
  int M, L;
};
__host__ __device__ inline int64_t tiles_at(int64_t M) { return 64 + (M + 3) / 4 * 4; }  // (16-byte aligned)

// Tile `no` as a wavefront sees it: its adapter, how many rows (0: no such tile), and the row in a slot (a row of the batch for an empty slot too).
struct Tile {
  int adapter = 0, rows = 0;
  int own;  // without a plan: lane s has the row in slot s
  const int32_t* order;
  __device__ __forceinline__ Tile(const Rows& r, int no, int lane) {
    if (r.plan) {
      order = nullptr, own = 0;
      if (no >= r.plan[0]) return;
      const RowTile t = ((const RowTile*)(r.plan + tiles_at(r.M)))[no];
      adapter = __builtin_amdgcn_readfirstlane(t.adapter), rows = __builtin_amdgcn_readfirstlane(t.rows);
      order = r.plan + 64 + __builtin_amdgcn_readfirstlane(t.first);
      return;
    }
    // row `no` begins a tile if a multiple of 16 rows of its adapter come before it
    int key = lane < r.M ? r.ids[lane] : -1;
    if ((uint32_t)key >= (uint32_t)r.L) key = r.L;
    const int mine = __builtin_amdgcn_readlane(key, no);
    const uint64_t same = __builtin_amdgcn_ballot_w64(lane < r.M && key == mine);
    const int before = __builtin_popcountll(same & (((uint64_t)1 << no) - 1));
    if (before % 16) return;
    const int place = __builtin_popcountll(same & (((uint64_t)1 << lane) - 1)) - before;
    const bool in = ((same >> lane) & 1) && place >= 0 && place < 16;
    own = __builtin_amdgcn_ds_permute(4 * (in ? place : 63), lane);  // (slots that nobody sends a row get row 0; lane 63's is nobody's slot)
    const int left = __builtin_popcountll(same) - before;
    adapter = mine, rows = left < 16 ? left : 16;
  }
  __device__ __forceinline__ int row(const Rows& r, int slot) const { return r.plan ? order[slot < rows ? slot : rows - 1] : __shfl(own, slot); }
};

// One work-group.  Rows are counted by adapter, every adapter's are cut into tiles of 2^tile_shift, and the rows take their places: a run of one adapter with
// one atomic addition a wavefront.  Which place of its adapter's a row gets may differ between runs; no value depends on it.  ONCE: up to AHEAD rows a
// lane, whose ids and places stay in registers.
template <bool ONCE, int THREADS, int AHEAD>
__global__ __launch_bounds__(THREADS) void low_rank_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ plan, int M, int L, int tile_shift) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int32_t count[kMaxAdapters + 1];
  __shared__ int32_t part[WAVES][2];
  const int tile_rows = 1 << tile_shift;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int id[AHEAD], place[AHEAD];
  const auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (r0 + i * THREADS >= M) break;
      const int r = r0 + i * THREADS + tid;
      id[i] = ids[r < M ? r : M - 1];
    }
  };
  const auto add = [&](int key, bool there) __attribute__((always_inline)) {  // -> the place among the rows counted so far
    const int first = __builtin_amdgcn_readfirstlane(key);
    const uint64_t live = __builtin_amdgcn_ballot_w64(there);
    if (__builtin_amdgcn_ballot_w64(there && key == first) == live && (live & 1)) {  // (rows that are there are the first lanes')
      int base = 0;
      if (lane == 0) base = atomicAdd(&count[first], __builtin_popcountll(live));
      return __builtin_amdgcn_readfirstlane(base) + lane;
    }
    return there ? atomicAdd(&count[key], 1) : 0;
  };
  const auto place_all = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (r0 + i * THREADS >= M) break;
      id[i] = (uint32_t)id[i] < (uint32_t)L ? id[i] : L;
      place[i] = add(id[i], r0 + i * THREADS + tid < M);
    }
  };
  if (ONCE) load(0);
  for (int i = tid; i <= L; i += THREADS) count[i] = 0;
  __syncthreads();
  for (int r0 = 0; r0 < M; r0 += THREADS * AHEAD) {
    if (!ONCE) load(r0);
    place_all(r0);
  }
  __syncthreads();
  // where every adapter's rows and tiles begin: neighbouring adapters a lane
  const int per = (L + THREADS) / THREADS;
  int rows = 0, tiles = 0;
  for (int i = 0; i < per; ++i) {
    const int n = tid * per + i <= L ? count[tid * per + i] : 0;
    rows += n, tiles += (n + tile_rows - 1) >> tile_shift;
  }
  int rows_to = rows, tiles_to = tiles;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(rows_to, o), b = __shfl_up(tiles_to, o);
    if (lane >= o) rows_to += a, tiles_to += b;
  }
  if (lane == 63) part[wave][0] = rows_to, part[wave][1] = tiles_to;
  __syncthreads();
  int row = rows_to - rows, tile = tiles_to - tiles;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) row += w < wave ? part[w][0] : 0, tile += w < wave ? part[w][1] : 0;
  RowTile* const out = (RowTile*)(plan + tiles_at(M));
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e > L) break;
    const int n = count[e];
    for (int at = 0; at < n; at += tile_rows) out[tile++] = RowTile{e, row + at, n - at < tile_rows ? n - at : tile_rows, 0};
    count[e] = row;
    row += n;
    if (e == L) plan[0] = tile;
  }
  __syncthreads();
  for (int r0 = 0; r0 < M; r0 += THREADS * AHEAD) {
    if (!ONCE) {
      load(r0);
      place_all(r0);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int r = r0 + i * THREADS + tid;
      if (r < M) plan[64 + place[i] + (ONCE ? count[id[i]] : 0)] = r;
    }
  }
}

// ---- the first product: sums[part][row][i] of h, parts of K -----------------------------------------------------------------
struct DownArgs {
  Rows r;
  const void *X, *A;
  float* sums;
  int K, rows, part_k;  // rows: of an adapter's A; part_k: values of a part, a multiple of 64 (tiles of 16 rows: of kDownStep)
  int groups, total;    // groups of rows of A of a tile, and tiles (runs of 16 rows of them)
  int subs;             // runs of 16 rows of a tile
};
// Work-group `no`: which of its tile's groups, and which tile.  (Numbers go to the XCDs in turn: the groups of a tile one after another on one of them.)
struct DownPlace {
  int group, tile;
  __device__ __forceinline__ DownPlace(int no, int groups) {
    const int turn = no >> 3;
    group = turn % groups, tile = (turn / groups) * 8 + (no & 7);
  }
};

// Tiles of 16 rows, or a tile of 64 in four runs, x 16 rows of A on one part of K: eight wavefronts take stages of 64 values (128 bytes, a cache line, of a row) in
// turn, each with a ring of its own in LDS, which it fills two stages ahead, eight lanes a line, and nobody else looks at; the wavefronts' sums meet at the end.  Operands read
// straight from memory -- 16 neighbouring lanes, 16 rows -- go through the cache at a quarter of its rate (13 bytes a clock and CU).  Whole calls, us, that
// way / this: 512 rows of 128 adapters 21.2 / 18.4, 259 of 32 of rank 64 on 2 x 11008 44.1 / 41.2; four wavefronts, or four stages ahead: level to 0.2 behind.
constexpr int kDownWaves = 8, kDownStep = 64 * kDownWaves;
template <typename T>
__global__ __launch_bounds__(64 * kDownWaves) void low_rank_down_kernel(const DownArgs a) {
  typedef typename MmaOf<T>::type Mma;
  constexpr int WAVES = kDownWaves, DEPTH = 2, LOADS = 4;
  __shared__ uint4_t stages[WAVES][DEPTH][32][8];
  __shared__ float4_t red[WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const DownPlace at(blockIdx.x, a.groups);
  const Tile tile(a.r, at.tile / a.subs, lane);
  const int slot0 = at.tile % a.subs * 16, live = tile.rows - slot0;
  if (at.tile >= a.total || live <= 0 || tile.adapter == a.r.L) return;
  const int part = blockIdx.y, col0 = at.group * 16, line = lane >> 3, chunk = (lane & 7) ^ line;
  const T* src[LOADS];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int col = col0 + i * 8 + line;
    src[i] = (const T*)a.X + (int64_t)tile.row(a.r, slot0 + i * 8 + line) * a.K;
    src[2 + i] = (const T*)a.A + ((int64_t)tile.adapter * a.rows + (col < a.rows ? col : a.rows - 1)) * a.K;
  }
  const int begin = part * a.part_k, end = begin + a.part_k < a.K ? begin + a.part_k : a.K;
  const int all = (end - begin + 63) / 64, steps = (all - wave + WAVES - 1) / WAVES;  // (this wavefront's: wave, wave + WAVES ..)
  const uint32_t lds = lds_of(stages[wave]);
  const auto load = [&](int s) __attribute__((always_inline)) {
    int k = begin + (s * WAVES + wave) * 64 + chunk * 8;
    k = k < a.K ? k : a.K - 8;  // (rows are multiples of 32 values: the second half of the last stage may not be there)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) direct16(src[i] + k, lds + (uint32_t)((s % DEPTH) * 4096 + i * 1024));
  };
  float4_t acc = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < DEPTH; ++s)
    if (s < steps) load(s);
  for (int s = 0; s < steps; ++s) {
    if (s + DEPTH <= steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint4_t(*const stage)[8] = stages[wave][s % DEPTH];
    const int k = begin + (s * WAVES + wave) * 64;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && k + 32 >= a.K) break;
      const int place = (half * 4 + q) ^ (r16 & 7);
      acc = Mma::mma(stage[16 + r16][place], stage[r16][place], acc);
    }
    if (s + DEPTH < steps) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      load(s + DEPTH);
    }
  }
  red[wave][lane] = acc;
  __syncthreads();
  const int i = col0 + q * 4;
  if (wave != 0 || r16 >= live || i >= a.rows) return;
#pragma unroll
  for (int v = 1; v < WAVES; ++v) acc += red[v][lane];
  *(float4_t*)(a.sums + (part * (int64_t)a.r.M + tile.row(a.r, slot0 + r16)) * a.rows + i) = acc;
}

// Tiles of 64 rows x 16 NT rows of A: rows and weights come in stages of 64 values (128 bytes, a cache line, of a row), eight lanes a line, straight into
// LDS, three stages ahead; a wavefront multiplies 16 rows.  8192 rows, K = 4096, rank 32 bf16: 16 us where X is in the last-level
// cache, 27 behind a second product that has just written 235 MB; five, seven stages ahead level.
template <typename T, int NT>
__global__ __launch_bounds__(256) void low_rank_down_tile_kernel(const DownArgs a) {
  typedef typename MmaOf<T>::type Mma;
  constexpr int DEPTH = 4, LINES = 64 + 16 * NT, W_LOADS = NT == 1 ? 1 : NT / 2, LOADS = 2 + W_LOADS;  // rows of a stage; loads of a wavefront
  __shared__ uint4_t stages[DEPTH][LINES][8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const DownPlace at(blockIdx.x, a.groups);
  const Tile tile(a.r, at.tile, lane);
  if (at.tile >= a.total || tile.rows == 0 || tile.adapter == a.r.L) return;
  const int part = blockIdx.y, col0 = at.group * 16 * NT;
  // chunk c of line r lies at place c ^ (r & 7): eight lines' chunks meet every bank once
  const int line = lane >> 3, chunk = (lane & 7) ^ line;
  const T* src[LOADS];
  uint32_t to[LOADS];
#pragma unroll
  for (int i = 0; i < 2; ++i) src[i] = (const T*)a.X + (int64_t)tile.row(a.r, wave * 16 + i * 8 + line) * a.K, to[i] = (wave * 16 + i * 8) * 128;
#pragma unroll
  for (int i = 0; i < W_LOADS; ++i) {
    const int first = (NT == 1 ? wave & 1 : wave * W_LOADS + i) * 8, col = col0 + first + line;  // (NT = 1: two wavefronts bring the same)
    src[2 + i] = (const T*)a.A + ((int64_t)tile.adapter * a.rows + (col < a.rows ? col : a.rows - 1)) * a.K, to[2 + i] = (64 + first) * 128;
  }
  const uint32_t lds = lds_of(stages);
  const int begin = part * a.part_k, end = begin + a.part_k < a.K ? begin + a.part_k : a.K, steps = (end - begin + 63) / 64;
  const auto load = [&](int s) __attribute__((always_inline)) {
    int k = begin + s * 64 + chunk * 8;
    k = k < a.K ? k : a.K - 8;  // (rows are multiples of 32 values: the second half of the last stage may not be there)
    const uint32_t stage = lds + (uint32_t)((s % DEPTH) * (LINES * 128));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) direct16(src[i] + k, stage + to[i]);
  };
  float4_t acc[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) acc[u] = float4_t{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < DEPTH - 1; ++s)
    if (s < steps) load(s);
  for (int s = 0; s < steps; ++s) {
    // this wavefront's loads of stage s have landed (DEPTH - 2 stages follow it; at the end all have), then everybody's, and nobody reads stage s - 1 any more
    if (s + DEPTH - 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((DEPTH - 2) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + DEPTH - 1 < steps) load(s + DEPTH - 1);
    const uint4_t(*const stage)[8] = stages[s % DEPTH];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && begin + s * 64 + 32 >= a.K) break;
      const int place = (half * 4 + q) ^ (r16 & 7);
      const uint4_t x = stage[wave * 16 + r16][place];
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[u] = Mma::mma(stage[64 + u * 16 + r16][place], x, acc[u]);
    }
  }
  if (wave * 16 + r16 >= tile.rows) return;
  float* const out = a.sums + (part * (int64_t)a.r.M + tile.row(a.r, wave * 16 + r16)) * a.rows;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int i = col0 + u * 16 + q * 4;
    if (i < a.rows) *(float4_t*)(out + i) = acc[u];
  }
}

// ---- the second product, and the sum -----------------------------------------------------------------------------------------
struct UpArgs {
  Rows r;
  const void *Y, *B;
  const float *scaling, *sums;
  void* out;
  int N, rows, parts;            // rows: of an adapter's A; parts: of K
  int end0, end1;                // where the first and the second part of the outputs end
  int per_group;                 // blocks of 128 outputs of a work-group
  int groups, groups0, groups1;  // work-groups of a tile: all, those ahead of the second part of the outputs and of the third
};

// Pieces of the operands' type for a value of h: one would round h to it, as much error as the output's own rounding.  Two of bfloat16 hold 16 of its 24 bits, 2^-8 of a
// step of the 16-bit output; three all of them, for an output in fp32 (8192 rows of rank 32 on 14336 outputs: 271 us either way; with a 16-bit output 139 / 146, of
// rank 64 150 / 170).  Two of float16 hold 22, of h times a power of two that brings the row's largest to 2^14 or above, below 2^15 (h itself may lie outside of float16's
// range).  float16's steps end at 2^-24, so its second piece is what the first leaves over times kPieceStep (2^15 at most again), with a sum of products of its own that
// is divided by that: values down to 2^-29 of the row's largest have 22 bits, smaller ones are off by 2^-51 of the largest.  (Without the step, the same rows take
// 145 us, with it 141; 500 rows of 40 adapters on 4096 outputs 16.5 / 16.7.)  (Beside an infinity the further pieces are 0.)
template <typename T, typename TO>
constexpr int kPieces = std::is_same<T, half_t>::value || sizeof(TO) == 2 ? 2 : 3;
constexpr float kPieceStep = 4096.0f;
__device__ __forceinline__ float rest(float h, float piece) { return fabsf(piece) < __builtin_inff() ? h - piece : 0.0f; }
template <typename T, int PIECES>
__device__ __forceinline__ void pieces_of(float (&h)[8], uint4_t (&piece)[PIECES]) {
#pragma unroll
  for (int n = 0; n < PIECES; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float first, second;
      if constexpr (std::is_same<T, half_t>::value) {
        const half2_t p = {(half_t)h[2 * i], (half_t)h[2 * i + 1]};
        piece[n][i] = bitcast<uint32_t>(p), first = (float)p[0], second = (float)p[1];
      } else {
        piece[n][i] = pack_bf16x2(h[2 * i], h[2 * i + 1]);
        first = bitcast<float>(piece[n][i] << 16), second = bitcast<float>(piece[n][i] & 0xffff0000u);
      }
      h[2 * i] = rest(h[2 * i], first), h[2 * i + 1] = rest(h[2 * i + 1], second);
      if constexpr (std::is_same<T, half_t>::value) h[2 * i] *= kPieceStep, h[2 * i + 1] *= kPieceStep;
    }
}

// Blocks of 128 outputs of one part of the outputs x 16 RW rows: RW wavefronts have 16 rows each and share a block's rows of B, 4 / RW (2: see kUpWaves)
// blocks go at a time.  A block of B, RANK values a row, comes into LDS in whole cache lines; output n = 8 r + j belongs to column r of the j-th of eight
// products of 16 x 16, so that 16 neighbouring lanes have 128 neighbouring outputs of one row of Y and out, 16 bytes each.
template <int RW, int RANK>
constexpr int kUpWaves = RW == 1 && RANK >= 64 ? 2 : 4;  // (32 KB of B for each wavefront)
template <typename T, typename TO, int RW, int RANK>
__global__ __launch_bounds__((64 * kUpWaves<RW, RANK>)) void low_rank_up_kernel(const UpArgs a) {
  typedef typename MmaOf<T>::type Mma;
  constexpr int CW = kUpWaves<RW, RANK> / RW, C = RANK / 8, RB = (RANK + 31) / 32, W = sizeof(TO) / 2, B_LOADS = 2 * C;  // chunks of a row of B, ..
  __shared__ uint4_t tiles[CW][128 * C];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4, rw = wave % RW, cw = wave / RW;
  // (work-groups that run at a time have neighbouring outputs of the same rows)
  const int at = blockIdx.x / a.groups, no = blockIdx.x - at * a.groups;
  const Tile tile(a.r, at, lane);
  if (tile.rows == 0) return;
  const bool with = tile.adapter != a.r.L;
  if (!with && a.Y == a.out) return;
  const int live = tile.rows - rw * 16;  // rows of this wavefront, if any
  int64_t row[4];                        // rows 4 q + i of its 16
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = tile.row(a.r, rw * 16 + q * 4 + i);
  const int p = (no >= a.groups0) + (no >= a.groups1), begin = p == 0 ? 0 : p == 1 ? a.end0 : a.end1, end = p == 0 ? a.end0 : p == 1 ? a.end1 : a.N;
  const int group = no - (p == 0 ? 0 : p == 1 ? a.groups0 : a.groups1);
  // line l of a block in LDS is its row 8 (l % 16) + l / 16; chunk c of it lies at place c ^ turn(l): eight lines' chunks meet every bank once
  const auto turn = [](int l) __attribute__((always_inline)) { return C == 1 ? 0 : C == 2 ? (l >> 2) & 1 : C == 4 ? (l >> 1) & 3 : l & 7; };
  const T* const b0 = (const T*)a.B + ((int64_t)tile.adapter * a.N + begin) * RANK;
  const uint32_t lds = lds_of(tiles[cw]);
  constexpr int PIECES = kPieces<T, TO>;
  uint4_t pieces[RB][PIECES];
  float back[4];  // the scaling, times what the pieces' power of two takes back, of rows 4 q + i
  for (int i = 0; i < a.per_group; i += CW) {
    const int n0 = (group * a.per_group + i + cw) * 128;
    if (begin + n0 >= end) break;
    if (with) {
      // (nobody reads the last block any more)
      if (i > 0) {
        if constexpr (RW > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int k = 0; k < (B_LOADS + RW - 1) / RW; ++k) {
        const int load = k * RW + rw;
        if (B_LOADS % RW != 0 && load >= B_LOADS) break;
        const int l = (load * 64 + lane) / C, c = lane % C ^ turn(l);
        int n = n0 + 8 * (l & 15) + (l >> 4);
        n = n < end - begin ? n : end - begin - 1;
        direct16(b0 + (int64_t)n * RANK + c * 8, lds + load * 1024);
      }
    }
    const int n = begin + n0 + r16 * 8;
    uint4_t y[4][W];
    if (n < end) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (q * 4 + m < live)
#pragma unroll
          for (int v = 0; v < W; ++v) y[m][v] = __builtin_nontemporal_load((const uint4_t*)((const TO*)a.Y + row[m] * a.N + n) + v);
    }
    if (with) {
      if (i == 0) {
        float h[RB][8];
        const float* s = a.sums + (int64_t)tile.row(a.r, rw * 16 + r16) * a.rows + p * RANK + q * 8;
        const int64_t step = (int64_t)a.r.M * a.rows;
#pragma unroll
        for (int c = 0; c < RB; ++c)
#pragma unroll
          for (int k = 0; k < 8; ++k) h[c][k] = 0.0f;
        if (RANK >= 32 || q < C) {
          constexpr int ONCE = RB == 1 ? 8 : 2;  // parts that are asked for at once
          for (int part = 0; part < a.parts; part += ONCE) {
            float4_t u[ONCE][RB], v[ONCE][RB];
#pragma unroll
            for (int o = 0; o < ONCE; ++o) {
              const float* const from = s + (part + o < a.parts ? part + o : part) * step;
#pragma unroll
              for (int c = 0; c < RB; ++c) u[o][c] = *(const float4_t*)(from + c * 32), v[o][c] = *(const float4_t*)(from + c * 32 + 4);
            }
#pragma unroll
            for (int o = 0; o < ONCE; ++o) {
              if (part + o >= a.parts) break;
#pragma unroll
              for (int c = 0; c < RB; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) h[c][k] += u[o][c][k], h[c][4 + k] += v[o][c][k];
            }
          }
        }
        float scale = a.scaling[tile.adapter];
        if constexpr (std::is_same<T, half_t>::value) {
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(h[c][k]));
          top = fmaxf(top, __shfl_xor(top, 16)), top = fmaxf(top, __shfl_xor(top, 32));
          // 2^e <= top < 2^(e + 1), e from -100 to 127 (a sum of products of float16 is 0 or 2^-48 at least; infinities and NaN stay what they are)
          int e = (int)(bitcast<uint32_t>(top) >> 23) - 127;
          e = e < -100 ? -100 : e > 127 ? 127 : e;
          const float down = bitcast<float>((uint32_t)(127 + 14 - e) << 23), up = bitcast<float>((uint32_t)(127 - 14 + e) << 23);
          scale *= up;
#pragma unroll
          for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) h[c][k] *= down;
        }
#pragma unroll
        for (int c = 0; c < RB; ++c) pieces_of<T>(h[c], pieces[c]);
#pragma unroll
        for (int m = 0; m < 4; ++m) back[m] = __shfl(scale, q * 4 + m);
      }
      if constexpr (RW > 1) asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      float4_t acc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[j] = float4_t{0, 0, 0, 0};
        float4_t less = {0, 0, 0, 0};  // (float16: of the second pieces)
#pragma unroll
        for (int c = 0; c < RB; ++c) {
          // (a rank below 32: the lanes behind it have zeros for h, and a chunk of the same row of B)
          const uint4_t b = tiles[cw][(j * 16 + r16) * C + ((C >= 4 ? c * 4 + q : q & (C - 1)) ^ turn(r16))];
#pragma unroll
          for (int of = PIECES - 1; of > 0; --of) {
            if constexpr (std::is_same<T, half_t>::value) less = Mma::mma(pieces[c][of], b, less);
            else acc[j] = Mma::mma(pieces[c][of], b, acc[j]);
          }
          acc[j] = Mma::mma(pieces[c][0], b, acc[j]);
        }
        if constexpr (std::is_same<T, half_t>::value)
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[j][m] = __builtin_fmaf(less[m], 1.0f / kPieceStep, acc[j][m]);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if constexpr (sizeof(TO) == 4) {
#pragma unroll
          for (int v = 0; v < W; ++v) {
            float4_t f = bitcast<float4_t>(y[m][v]);
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = __builtin_fmaf(back[m], acc[4 * v + k][m], f[k]);
            y[m][v] = bitcast<uint4_t>(f);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t two = y[m][0][k];
            float f[2];
            if constexpr (std::is_same<T, half_t>::value) f[0] = (float)bitcast<half2_t>(two)[0], f[1] = (float)bitcast<half2_t>(two)[1];
            else f[0] = bitcast<float>(two << 16), f[1] = bitcast<float>(two & 0xffff0000u);
            f[0] = __builtin_fmaf(back[m], acc[2 * k][m], f[0]), f[1] = __builtin_fmaf(back[m], acc[2 * k + 1][m], f[1]);
            if constexpr (std::is_same<T, half_t>::value) y[m][0][k] = bitcast<uint32_t>(half2_t{(half_t)f[0], (half_t)f[1]});
            else y[m][0][k] = pack_bf16x2(f[0], f[1]);
          }
        }
      }
    }
    if (n < end) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (q * 4 + m < live)
#pragma unroll
          for (int v = 0; v < W; ++v) *((uint4_t*)((TO*)a.out + row[m] * a.N + n) + v) = y[m][v];
    }
  }
}

// ---- single rows: both products in one launch ---------------------------------------------------------------------------------
struct RowArgs {
  const int32_t* ids;
  const void *X, *Y, *A, *B;
  const float* scaling;
  void* out;
  int L, N, K, rows, end0, end1;  // as above
  int per_group, groups, groups0, groups1, M;
};
template <typename T>
__device__ __forceinline__ float value8(const uint4_t& v, int k) {
  if constexpr (std::is_same<T, half_t>::value) return (float)bitcast<half2_t>(v[k / 2])[k % 2];
  else return bitcast<float>(k % 2 ? v[k / 2] & 0xffff0000u : v[k / 2] << 16);
}

// A row and blocks of 4096 / RANK outputs of one part of the outputs a work-group, which forms the part's RANK values of h for itself: CL lanes have a run of
// 8 CL values of each of H rows of A, the wavefronts take K in turn, and their sums meet in LDS; X, A and the first four blocks' B and Y are asked for at once.
// Bounded by latency and by A through the CU (rank 16, K = 4096: 128 KB, about 1 us of 3.9).  More code costs more than loads it has in flight: a row of rank 8,
// K = 4096, with 8 / 16 / 32 loads of A at a time 3.3 / 3.9 / 5.3 us; sixteen wavefronts 4.6.  CL = 16 reads X less often, 8 has fewer sums a lane, us, 16 / 8: rank
// 32 5.9 / 5.1, 64 10.6 / 7.9, 8, K = 11008, 4.7 / 5.2.  One / two / four / eight blocks at a time (work-groups spread over the XCDs): 16 rows of
// rank 16 on 22016 outputs 9.7 / 8.0 / 7.4 / 7.2, 64 of 48 adapters on 6144 11.0 / 9.2 / 8.6 / 8.5, 16 of rank 32 on 14336 11.8 / 10.1 / 9.4 / 10.5.
constexpr int kRowWaves = 8;
// From so many rows on a row's work-groups go to one XCD, whose L2 reads the row's A once; fewer would leave XCDs without work.  Spread / together, us, rank 16, K = 4096:
// 4 rows on 22016 outputs 4.2 / 6.0, 8 5.3 / 4.8, 8 on 4096 4.0 / 4.2, 32 7.0 / 5.0, 64 of 48 adapters on 6144 8.5 / 7.3; rank 8, K = 11008, 64 9.5 / 6.2.
constexpr int kTogether = 8;
template <typename T, typename TO, int RANK>
__global__ __launch_bounds__(64 * kRowWaves) void low_rank_row_kernel(const RowArgs a) {
  constexpr int WAVES = kRowWaves, CL = RANK >= 32 ? 8 : 16, LINES = 64 / CL, STAGE = CL * 8, H = RANK / LINES, AHEAD = 8 / H, BLOCKS = 4;
  static_assert(H <= 8 && H <= CL, "the sums of a run of lanes end as one a lane");
  constexpr int C = RANK / 8, OUT = 64 * WAVES / C;  // chunks of a row of B, outputs of a block
  __shared__ float4_t sums[WAVES][RANK / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int row = blockIdx.x / a.groups, no = blockIdx.x - row * a.groups;
  if (a.M >= kTogether) {
    const DownPlace at(blockIdx.x, a.groups);
    row = at.tile, no = at.group;
    if (row >= a.M) return;
  }
  const int p = (no >= a.groups0) + (no >= a.groups1), begin = p == 0 ? 0 : p == 1 ? a.end0 : a.end1, end = p == 0 ? a.end0 : p == 1 ? a.end1 : a.N;
  const int first = begin + (no - (p == 0 ? 0 : p == 1 ? a.groups0 : a.groups1)) * a.per_group * OUT, n_end = end - first < a.per_group * OUT ? end - first : a.per_group * OUT;
  const int adapter = a.ids[row];
  const TO* const y_row = (const TO*)a.Y + (int64_t)row * a.N + first;
  TO* const out_row = (TO*)a.out + (int64_t)row * a.N + first;
  if ((uint32_t)adapter >= (uint32_t)a.L) {
    if (a.Y != a.out)
      for (int n = tid; n < n_end; n += 64 * kRowWaves) out_row[n] = y_row[n];
    return;
  }
  const uint4_t* const b_row = (const uint4_t*)((const T*)a.B + ((int64_t)adapter * a.N + first) * RANK);
  const int place = tid % C;
  uint4_t b[BLOCKS];
  TO y[BLOCKS];
  const auto load = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      if (n0 + u * OUT >= n_end) break;
      int n = n0 + u * OUT + tid / C;
      n = n < n_end ? n : n_end - 1;
      b[u] = b_row[(int64_t)n * C + place], y[u] = y_row[n];
    }
  };
  load(0);
  const float scale = a.scaling[adapter];
  const int chunk = lane % CL, line = lane / CL;
  const T* const x = (const T*)a.X + (int64_t)row * a.K;
  const T* const w = (const T*)a.A + ((int64_t)adapter * a.rows + p * RANK + line) * a.K;
  float h[H];
#pragma unroll
  for (int j = 0; j < H; ++j) h[j] = 0.0f;
  for (int k0 = wave * STAGE + chunk * 8; k0 - chunk * 8 < a.K; k0 += AHEAD * STAGE * WAVES) {
    uint4_t xs[AHEAD], ws[AHEAD][H];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * STAGE * WAVES < a.K ? k0 + u * STAGE * WAVES : a.K - 8;
      xs[u] = *(const uint4_t*)(x + k);
#pragma unroll
      for (int j = 0; j < H; ++j) ws[u][j] = *(const uint4_t*)(w + (int64_t)j * LINES * a.K + k);
    }
    asm volatile("" ::: "memory");  // (all loads ahead of the first value's use)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (k0 + u * STAGE * WAVES >= a.K) break;
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) h[j] = __builtin_fmaf(value8<T>(xs[u], k), value8<T>(ws[u][j], k), h[j]);
    }
  }
  // sums over a run's lanes: of two values a lane has, it keeps one and hands over the other, while there are two
  int at = 0;
#pragma unroll
  for (int o = CL / 2, n = H; o >= 1; o /= 2) {
    if (n > 1) {
      n /= 2;
      const bool upper = chunk & o;
      at += upper ? n : 0;
#pragma unroll
      for (int j = 0; j < H / 2; ++j)
        if (j < n) h[j] = (upper ? h[j + n] : h[j]) + __shfl_xor(upper ? h[j] : h[j + n], o);
    } else {
      h[0] += __shfl_xor(h[0], o);
    }
  }
  ((float*)sums[wave])[at * LINES + line] = h[0];
  __syncthreads();
  float4_t low = sums[0][place * 2], high = sums[0][place * 2 + 1];
#pragma unroll
  for (int v = 1; v < WAVES; ++v) low += sums[v][place * 2], high += sums[v][place * 2 + 1];
  for (int n0 = 0; n0 < n_end; n0 += BLOCKS * OUT) {
    if (n0 > 0) load(n0);
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      if (n0 + u * OUT >= n_end) break;
      float f = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) f = __builtin_fmaf(value8<T>(b[u], k), low[k], f);
#pragma unroll
      for (int k = 0; k < 4; ++k) f = __builtin_fmaf(value8<T>(b[u], 4 + k), high[k], f);
#pragma unroll
      for (int o = 1; o < C; o *= 2) f += __shfl_xor(f, o);
      const int n = n0 + u * OUT + tid / C;
      if (place == 0 && n < n_end) {
        if constexpr (sizeof(TO) == 4) out_row[n] = __builtin_fmaf(scale, f, y[u]);
        else if constexpr (std::is_same<TO, half_t>::value) out_row[n] = (half_t)__builtin_fmaf(scale, f, (float)y[u]);
        else ((uint16_t*)out_row)[n] = (uint16_t)pack_bf16x2(__builtin_fmaf(scale, f, bitcast<float>((uint32_t)bitcast<uint16_t>(y[u]) << 16)), 0.0f);
      }
    }
  }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------
constexpr int64_t kMostGroups = ((int64_t)1 << 24) - 1;  // work-groups of 256 threads of a launch, which has fewer than 2^32 threads
inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
// Tiles of 64 rows where an adapter has 32 or more on average and B is large enough to be worth sharing: the work-groups of a tile of 64 read it once,
// those of 16 four times, and are twice as many.  Whole calls, us, K = 4096, tiles of 16 / 64 (first product by one_run_each): rank 16 on 4096 outputs, 1003 rows of 8
// adapters 17.5 / 17.7, 4000 33.6 / 36.0, 8000 63.2 / 62.9; rank 64, 500 of 12 26.0 / 26.6, 1003 24.9 / 23.3, 1003 on 14336 outputs 47.8 / 38.6; rank 32 on
// 14336, 8192 of 16 177 / 135.
inline int tile_rows_of(int64_t M, int64_t L, int64_t rank) { return M > kInlineRows && M >= 32 * L && M * rank >= 50000 ? 64 : 16; }
// Of tiles of 64 rows, the first product in runs of 16 (A read by each, but work-groups enough) or by whole tiles: 1003 rows, 64 rows of A 23.3 / 28.3, 128 28.6 /
// 33.9; 2000, 128 82.8 / 77.6; 8192, 16 65.2 / 67.0, 32 136.9 / 135.5, 64 88.6 / 78.3.
inline bool one_run_each(int64_t M, int64_t rows) { return M * rows <= 160000; }
inline int64_t most_tiles(int64_t M, int64_t L, int tile_rows) { return M <= kInlineRows ? M : M / tile_rows + (L + 1 < M ? L + 1 : M); }
int64_t plan_bytes(int64_t M, int64_t L) { return M <= kInlineRows ? 0 : align256((tiles_at(M) + 4 * most_tiles(M, L, 16)) * 4); }
// Parts of K: work-groups for the machine where there are few tiles (`want` of them), at most 16, or 4 for tiles of 16 rows, whose eight wavefronts share K
// already.  Every part costs a sum written and read: tiles of 64 rows: 8192 rows of rank 32 on 14336 outputs 136 us in one part, 139 in four, 145 in seven;
// 2048 of rank 16, three projections, 31.2 for 128 work-groups, 33.4 for 256; tiles of 16: 1 row of rank 32, K = 11008, 8.8 in two, 8.5 in
// four, 9.1 in eight, 9.7 in sixteen; 8 rows of rank 16, K = 28672, 13.2, 10.8, 10.5, 11.7.
// With more than M / 64 (M / 16) tiles, parts * M is less than 64 * kTileGroups + M (16 * kFewGroups + M).
constexpr int kTileGroups = 128, kFewGroups = 192, kFewParts = 4;
int64_t most_parts(int64_t K, int64_t most = 16) { return K >= 256 * most ? most : (K + 255) / 256; }
int64_t parts_of(int64_t tiles, int64_t K, int64_t want, int64_t most) {
  const int64_t parts = (want + tiles - 1) / tiles, can = most_parts(K, most);
  return parts < can ? parts : can;
}
int64_t sum_rows(int64_t M, int64_t K) {
  const int64_t few = most_parts(K) * M, many = 64 * kTileGroups + M;
  return few < many ? few : many;
}
static_assert(16 * kFewGroups <= 64 * kTileGroups, "sum_rows holds for both");

// Single rows where it is not too much that all work-groups of a row read its part of A (2 rank K bytes; there are up to N rank / 4096 of them) and all rows their
// adapter's B, which tiles share: neither a plan nor a second launch.  Whole calls, us, with them / this.  Rank 16: K = N = 4096, 1 row 7.0 / 3.9, 16 8.0 / 4.5; 64 of 48
// adapters on 6144 outputs 10.0 / 7.3, 52 of 200, K = 4352, on 19056 15.8 / 14.3, 47 of one on 22224 10.8 / 11.8; K = 736, 219 on 18352 14.2 / 20.8.  Rank 32: 22, K = 4672,
// on 9600 9.3 / 9.4, 27, K = 2976, on 16640 9.6 / 13.4.  Rank 64: 1 row, K = 2080, 7.4 / 6.0, 4, K = 1184, on 16832 7.8 / 7.8, K = 3392 8.5 / 10.1, 8, K = 3424,
// on 784 8.2 / 7.5.  Rank 128: 4, K = 512, on 2224 8.4 / 7.3, 2, K = 1312, on 2528 8.6 / 9.2: left to tiles.  Rank 8: K = 8000, 336 on 21104 28.9 / 27.4, K = 7360,
// 753 on 15248 24.8 / 21.7, K = 1568, 1977 on 13536 44.7 / 65.3; 256 -> 256, 5000 15.6 / 15.6, 64 -> 256, 10000 21.0 / 22.3.
// A bound on sizes alone, and not the best one: of these it takes the slower way, by 9 to 23 %, for the 47 rows of one adapter (tiles share its B; how many adapters the
// rows have is not among its arguments), for 1 and 8 rows of rank 64 with K = 2080 and 3424, for the 753 of rank 8 and, for want of that kernel, for the 4 of rank 128.
inline bool single_rows(int64_t M, int64_t rank, int64_t K, int64_t N) {
  return M <= 4096 && rank <= 64 && rank * K <= (int64_t)1 << 18 && rank * rank * K <= (int64_t)1 << 23 &&
         M * rank * rank * (K + N) <= (int64_t)(M <= kInlineRows ? 3 : 6) << 27;
}
// (384 / 256 / 192, spread over the XCDs: rank 16, 64 rows of 48 adapters on 6144 outputs 10.6 / 8.6 / 8.5, of one on 14336 7.2 / 7.2 / 9.4, 8 on 22016 6.7 / 5.3 / 5.5)
constexpr int kRowGroups = 256;

struct Call {
  Rows r;
  const void *X, *Y, *A, *B;
  const float* scaling;
  void* out;
  int32_t* plan;
  float* sums;
  int K, N, rank, rows, end0, end1;
};

// NT: 16 rows of A each that a work-group has; 0: runs of 16 rows, subs of them a tile
template <typename T, int NT>
int run_down(const Call& c, int64_t tiles, int subs, int64_t* parts, hipStream_t st) {
  const int groups = (c.rows + 16 * (NT ? NT : 1) - 1) / (16 * (NT ? NT : 1));
  // (an adapter's last tile is half empty on average, and so counts as half of one)
  const int64_t whole = NT ? tiles - (c.r.L + 1 < c.r.M ? c.r.L + 1 : c.r.M) / 2 : tiles * subs, step = NT ? 64 : kDownStep;
  const int part_k = (int)(ceil_div(ceil_div(c.K, parts_of(groups * whole, c.K, NT ? kTileGroups : kFewGroups, NT ? 16 : kFewParts)), step) * step);
  *parts = ceil_div(c.K, part_k);
  const DownArgs a{c.r, c.X, c.A, c.sums, c.K, c.rows, part_k, groups, (int)(tiles * subs), subs};
  const dim3 grid((unsigned)(ceil_div(tiles * subs, (int64_t)8) * 8 * groups), (unsigned)*parts);
  if constexpr (NT == 0) low_rank_down_kernel<T><<<grid, 64 * kDownWaves, 0, st>>>(a);
  else low_rank_down_tile_kernel<T, NT><<<grid, 256, 0, st>>>(a);
  return check_launch("tlq_low_rank_update", NT ? "low_rank_down_tile_kernel" : "low_rank_down_kernel") ? 0 : 1;
}

template <typename T, typename TO, int RW, int RANK>
int run_up(const Call& c, int64_t tiles, int64_t parts, hipStream_t st) {
  constexpr int WAVES = kUpWaves<RW, RANK>, CW = WAVES / RW;
  const int64_t blocks[3] = {(c.end0 + 127) / 128, (c.end1 - c.end0 + 127) / 128, (c.N - c.end1 + 127) / 128};
  const auto groups = [&](int per) { return ceil_div(blocks[0], (int64_t)per) + ceil_div(blocks[1], (int64_t)per) + ceil_div(blocks[2], (int64_t)per); };
  // h is made ready once a work-group: as many blocks for each as leave eight work-groups a CU (8192 rows of rank 32 on 14336 outputs bf16: 99 us; four a CU
  // 117, sixteen 101; 259 rows of rank 64 on 2 x 11008, the whole call: 43.7 / 46.2 / 47.7)
  int per_group = CW;
  while ((per_group < 32 && tiles * groups(per_group) > 2048) || tiles * groups(per_group) > kMostGroups) per_group += per_group < 32 ? CW : per_group;
  const int groups0 = (int)ceil_div(blocks[0], (int64_t)per_group), groups1 = groups0 + (int)ceil_div(blocks[1], (int64_t)per_group);
  const UpArgs a{c.r, c.Y, c.B, c.scaling, c.sums, c.out, c.N, c.rows, (int)parts, c.end0, c.end1, per_group, (int)groups(per_group), groups0, groups1};
  low_rank_up_kernel<T, TO, RW, RANK><<<(unsigned)(tiles * groups(per_group)), 64 * WAVES, 0, st>>>(a);
  return check_launch("tlq_low_rank_update", "low_rank_up_kernel") ? 0 : 1;
}
template <typename T, typename TO, int RW>
int run_up(const Call& c, int64_t tiles, int64_t parts, hipStream_t st) {
  switch (c.rank) {
    case 8: return run_up<T, TO, RW, 8>(c, tiles, parts, st);
    case 16: return run_up<T, TO, RW, 16>(c, tiles, parts, st);
    case 32: return run_up<T, TO, RW, 32>(c, tiles, parts, st);
    case 64: return run_up<T, TO, RW, 64>(c, tiles, parts, st);
    default: return run_up<T, TO, RW, 128>(c, tiles, parts, st);
  }
}

template <typename T, typename TO, int RANK>
int run_rows(const Call& c, hipStream_t st) {
  constexpr int OUT = 512 * kRowWaves / RANK;
  const int64_t blocks[3] = {(c.end0 + OUT - 1) / OUT, (c.end1 - c.end0 + OUT - 1) / OUT, (c.N - c.end1 + OUT - 1) / OUT};
  const auto groups = [&](int64_t per) { return ceil_div(blocks[0], per) + ceil_div(blocks[1], per) + ceil_div(blocks[2], per); };
  int per_group = 1;
  while (c.r.M * groups(per_group) > kRowGroups && per_group < 1 << 20) per_group *= 2;
  const int groups0 = (int)ceil_div(blocks[0], (int64_t)per_group), groups1 = groups0 + (int)ceil_div(blocks[1], (int64_t)per_group);
  const RowArgs a{c.r.ids, c.X, c.Y, c.A, c.B, c.scaling, c.out, c.r.L, c.N, c.K, c.rows, c.end0, c.end1, per_group, (int)groups(per_group), groups0, groups1, c.r.M};
  low_rank_row_kernel<T, TO, RANK><<<(unsigned)((c.r.M >= kTogether ? ceil_div(c.r.M, 8) * 8 : c.r.M) * groups(per_group)), 64 * kRowWaves, 0, st>>>(a);
  return check_launch("tlq_low_rank_update", "low_rank_row_kernel") ? 0 : 1;
}
template <typename T, typename TO>
int run_rows(const Call& c, hipStream_t st) {
  switch (c.rank) {
    case 8: return run_rows<T, TO, 8>(c, st);
    case 16: return run_rows<T, TO, 16>(c, st);
    case 32: return run_rows<T, TO, 32>(c, st);
    default: return run_rows<T, TO, 64>(c, st);
  }
}

template <typename T, typename TO>
int run_low_rank(Call c, hipStream_t st) {
  if (single_rows(c.r.M, c.rank, c.K, c.N)) return run_rows<T, TO>(c, st);
  const int tile_rows = tile_rows_of(c.r.M, c.r.L, c.rank);
  const int64_t tiles = most_tiles(c.r.M, c.r.L, tile_rows);
  int64_t parts = 1;
  if (c.r.M > kInlineRows) {
    const int shift = tile_rows == 16 ? 4 : 6;
    // (259 rows: four wavefronts 2.8 us, sixteen 4.4; 1003 level; 8192: sixteen 6.8, eight 8.5)
    if (c.r.M <= 1024) low_rank_plan_kernel<true, 256, 4><<<1, 256, 0, st>>>(c.r.ids, c.plan, c.r.M, c.r.L, shift);
    else if (c.r.M <= 8192) low_rank_plan_kernel<true, 1024, 8><<<1, 1024, 0, st>>>(c.r.ids, c.plan, c.r.M, c.r.L, shift);
    else low_rank_plan_kernel<false, 1024, 8><<<1, 1024, 0, st>>>(c.r.ids, c.plan, c.r.M, c.r.L, shift);
    if (!check_launch("tlq_low_rank_update", "low_rank_plan_kernel")) return 1;
    c.r.plan = c.plan;
  }
  const int rc = tile_rows == 16 ? run_down<T, 0>(c, tiles, 1, &parts, st)
                 : one_run_each(c.r.M, c.rows) ? run_down<T, 0>(c, tiles, 4, &parts, st)
                 : c.rows <= 16 ? run_down<T, 1>(c, tiles, 1, &parts, st)
                 : c.rows <= 32 ? run_down<T, 2>(c, tiles, 1, &parts, st)
                                : run_down<T, 4>(c, tiles, 1, &parts, st);
  if (rc) return rc;
  return tile_rows == 16 ? run_up<T, TO, 1>(c, tiles, parts, st) : run_up<T, TO, 4>(c, tiles, parts, st);
}

bool sizes_taken(int64_t M, int64_t L, int64_t rank, int64_t parts, int64_t K) {
  return M >= 0 && M < ((int64_t)1 << 24) && L >= 1 && L <= kMaxAdapters && (rank == 8 || rank == 16 || rank == 32 || rank == 64 || rank == 128) && parts >= 1 && parts <= 3 &&
         K >= 32 && K % 32 == 0 && K < ((int64_t)1 << 24);
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int64_t tlq_low_rank_update_workspace_bytes(int64_t M, int64_t L, int64_t rank, int64_t parts, int64_t K) {
  if (!sizes_taken(M, L, rank, parts, K)) return 0;
  return plan_bytes(M, L) + sum_rows(M, K) * parts * rank * 4;
}

extern "C" int tlq_low_rank_update(const void* X, const void* Y, const void* ids, const void* A, const void* B, const void* scaling, void* out,
                                   void* workspace, int64_t workspace_bytes, int64_t M, int64_t L, int64_t rank, int64_t n0, int64_t n1, int64_t n2,
                                   int64_t K, int in_dtype, int out_dtype, void* stream) {
  const char* const what = "tlq_low_rank_update";
  const int64_t parts = n1 == 0 ? 1 : n2 == 0 ? 2 : 3, N = n0 + n1 + n2;
  TLQ_REQUIRE(n0 >= 16 && n1 >= 0 && n2 >= 0 && (n1 > 0 || n2 == 0) && n0 % 16 == 0 && n1 % 16 == 0 && n2 % 16 == 0 && n0 < ((int64_t)1 << 24) &&
                  n1 < ((int64_t)1 << 24) && n2 < ((int64_t)1 << 24),
              "%s: parts must be multiples of 16, one to three of them (got %lld, %lld, %lld)", what, (long long)n0, (long long)n1, (long long)n2);
  TLQ_REQUIRE(sizes_taken(M, L, rank, parts, K),
              "%s: bad shape M=%lld L=%lld rank=%lld K=%lld (M below 2^24, 1 to 4096 adapters, rank 8, 16, 32, 64 or 128, K a multiple of 32)", what,
              (long long)M, (long long)L, (long long)rank, (long long)K);
  TLQ_REQUIRE(in_dtype == TLQ_F16 || in_dtype == TLQ_BF16, "%s: in_dtype must be float16 or bfloat16 (got %d)", what, in_dtype);
  TLQ_REQUIRE(out_dtype == in_dtype || out_dtype == TLQ_F32, "%s: out_dtype must be in_dtype or float32 (got %d)", what, out_dtype);
  if (M == 0) return 0;
  TLQ_REQUIRE(X && Y && ids && A && B && scaling && out, "%s: null pointer", what);
  TLQ_REQUIRE((((uintptr_t)X | (uintptr_t)Y | (uintptr_t)A | (uintptr_t)B | (uintptr_t)out) & 15) == 0 && (((uintptr_t)ids | (uintptr_t)scaling) & 3) == 0,
              "%s: X, Y, A, B and out must be 16-byte aligned, ids and scaling to their type", what);
  const int64_t want = tlq_low_rank_update_workspace_bytes(M, L, rank, parts, K);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && ((uintptr_t)workspace & 15) == 0, "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  const Call c{{(const int32_t*)ids, nullptr, (int)M, (int)L}, X, Y, A, B, (const float*)scaling, out, (int32_t*)workspace, (float*)((uint8_t*)workspace + plan_bytes(M, L)),
               (int)K, (int)N, (int)rank, (int)(parts * rank), (int)n0, (int)(n0 + n1)};
  hipStream_t st = (hipStream_t)stream;
  if (in_dtype == TLQ_F16) return out_dtype == TLQ_F32 ? run_low_rank<half_t, float>(c, st) : run_low_rank<half_t, half_t>(c, st);
  return out_dtype == TLQ_F32 ? run_low_rank<bf16_t, float>(c, st) : run_low_rank<bf16_t, bf16_t>(c, st);
}
