// Low-rank adapters of many requests beside a projection of up to three parts side by side (queries, keys, values; gate and up):
//   out[m, n] = rn(Y[m, n] + scaling[l] * sum_j h[m, p r + j] * B[l, n, j]),  h[m, i] = sum_k X[m, k] * A[l, i, k]
// l = ids[m], p the part that n lies in, r the rank; a row whose id names no adapter is out = Y.  h and the sums are fp32, rounded once, at the end.
//
// Memory bound: Y and out, X, and the weights of the adapters that some row names, each once.  Rows are gathered by adapter into tiles of 16 or 64, which
// meet their adapter's weights on the matrix units: the first product writes fp32 sums of parts of K (few tiles: many parts), the second adds the parts
// as it reads them.  A row's values do not depend on its tile or its place there.
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

// Tile `no` as a wavefront sees it: its adapter, how many rows (0: no such tile), and the row in slot s < 16 MT (a row of the batch for an empty slot too).
template <int MT>
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

// One work-group.  Rows are counted by adapter, every adapter's are cut into tiles of 64, and the rows take their places: a run of one adapter with one
// atomic addition a wavefront.  Which place of its adapter's a row gets may differ between runs; no value depends on it.
__global__ __launch_bounds__(1024) void low_rank_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ plan, int M, int L) {
  __shared__ int32_t count[kMaxAdapters + 1];
  __shared__ int32_t part[16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i <= L; i += 1024) count[i] = 0;
  __syncthreads();
  // f(row, its adapter or L, what the rows of the wavefront before it with the same adapter are if all of them have one, whether so, whether there is a row)
  const auto add = [&](int key, bool there) __attribute__((always_inline)) {  // -> the place among the rows counted so far
    const int first = __builtin_amdgcn_readfirstlane(key);
    const uint64_t live = __builtin_amdgcn_ballot_w64(there);
    if (__builtin_amdgcn_ballot_w64(there && key == first) == live && (live & 1)) {
      int base = 0;
      if (lane == 0) base = atomicAdd(&count[first], __builtin_popcountll(live));
      return __builtin_amdgcn_readfirstlane(base) + lane;
    }
    return there ? atomicAdd(&count[key], 1) : 0;
  };
  constexpr int AHEAD = 8;
  const auto each = [&](auto&& f) __attribute__((always_inline)) {
    for (int r0 = 0; r0 < M; r0 += 1024 * AHEAD) {
      int id[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = r0 + i * 1024 + tid;
        id[i] = ids[r < M ? r : M - 1];
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = r0 + i * 1024 + tid;
        f(r, (uint32_t)id[i] < (uint32_t)L ? id[i] : L, r < M);
      }
    }
  };
  each([&](int, int key, bool there) __attribute__((always_inline)) { add(key, there); });
  __syncthreads();
  // where every adapter's rows and tiles begin: five neighbouring adapters a lane
  constexpr int PER = (kMaxAdapters + 1024) / 1024;
  int rows = 0, tiles = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int n = tid * PER + i <= L ? count[tid * PER + i] : 0;
    rows += n, tiles += (n + 63) / 64;
  }
  int rows_to = rows, tiles_to = tiles;
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(rows_to, o), b = __shfl_up(tiles_to, o);
    if (lane >= o) rows_to += a, tiles_to += b;
  }
  if (lane == 63) part[wave][0] = rows_to, part[wave][1] = tiles_to;
  __syncthreads();
  int row = rows_to - rows, tile = tiles_to - tiles;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) row += part[w][0], tile += part[w][1];
  }
  RowTile* const out = (RowTile*)(plan + tiles_at(M));
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = tid * PER + i;
    if (e > L) break;
    const int n = count[e];
    for (int at = 0; at < n; at += 64) out[tile++] = RowTile{e, row + at, n - at < 64 ? n - at : 64, 0};
    count[e] = row;
    row += n;
    if (e == L) plan[0] = tile;
  }
  __syncthreads();
  each([&](int r, int key, bool there) __attribute__((always_inline)) {
    const int place = add(key, there);
    if (there) plan[64 + place] = r;
  });
}

// ---- the first product: sums[part][row][i] of h, parts of K -----------------------------------------------------------------
struct DownArgs {
  Rows r;
  const void *X, *A;
  float* sums;
  int K, rows, part_k;  // rows: of an adapter's A; part_k: values of a part, a multiple of 256
};

// 16 MT rows x 16 NT rows of A on one part of K, which the four wavefronts share out in steps of 64 values; both operands straight into registers.
template <typename T, int MT, int NT>
__global__ __launch_bounds__(256) void low_rank_down_kernel(const DownArgs a) {
  typedef typename MmaOf<T>::type Mma;
  __shared__ float4_t red[4][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const Tile<MT> tile(a.r, blockIdx.x, lane);
  if (tile.rows == 0 || tile.adapter == a.r.L) return;
  const int part = blockIdx.y, col0 = blockIdx.z * 16 * NT, frags = (tile.rows + 15) / 16;
  int row[MT];
  const T *x[MT], *w[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) row[t] = tile.row(a.r, t * 16 + r16), x[t] = (const T*)a.X + (int64_t)row[t] * a.K + q * 8;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int i = col0 + t * 16 + r16;
    w[t] = (const T*)a.A + ((int64_t)tile.adapter * a.rows + (i < a.rows ? i : a.rows - 1)) * a.K + q * 8;
  }
  float4_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = float4_t{0, 0, 0, 0};
  const int end = (part + 1) * a.part_k < a.K ? (part + 1) * a.part_k : a.K;
  for (int k = part * a.part_k + wave * 64; k < end; k += 256) {
    const bool both = k + 32 < a.K;  // (rows are multiples of 32 values)
    uint4_t wf[NT][2], xf[MT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      wf[u][0] = *(const uint4_t*)(w[u] + k);
      wf[u][1] = both ? *(const uint4_t*)(w[u] + k + 32) : uint4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t >= frags) break;
      xf[t][0] = *(const uint4_t*)(x[t] + k);
      xf[t][1] = both ? *(const uint4_t*)(x[t] + k + 32) : uint4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t >= frags) break;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        acc[t][u] = Mma::mma(wf[u][0], xf[t][0], acc[t][u]);
        acc[t][u] = Mma::mma(wf[u][1], xf[t][1], acc[t][u]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) red[wave][t * NT + u][lane] = acc[t][u];
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int f = t * NT + u, i = col0 + u * 16 + q * 4;
      if (f % 4 != wave || t * 16 + r16 >= tile.rows || i >= a.rows) continue;
      const float4_t sum = (red[0][f][lane] + red[1][f][lane]) + (red[2][f][lane] + red[3][f][lane]);
      *(float4_t*)(a.sums + ((int64_t)part * a.r.M + row[t]) * a.rows + i) = sum;
    }
}

// ---- the second product, and the sum -----------------------------------------------------------------------------------------
struct UpArgs {
  Rows r;
  const void *Y, *B;
  const float *scaling, *sums;
  void* out;
  int N, rank, rows, parts;  // rows: of an adapter's A; parts: of K
  int end0, end1;            // where the first and the second part of the outputs end
  int per_group;             // blocks of 64 outputs of a work-group
};

// Two pieces of the operands' type for a value of h: bfloat16 holds 16 of its bits that way; float16 22, of h over a power of two that brings the row's
// largest below 2 (h itself may lie outside of float16's range).  One piece would round h to the operands' type: as much error as the output's own rounding.
// (Beside an infinity the second piece is 0.)
__device__ __forceinline__ float rest(float h, float piece) { return fabsf(piece) < __builtin_inff() ? h - piece : 0.0f; }
template <typename T>
__device__ __forceinline__ void two_pieces(const float (&h)[8], uint4_t& high, uint4_t& low) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, half_t>::value) {
      const half2_t p = {(half_t)h[2 * i], (half_t)h[2 * i + 1]};
      high[i] = bitcast<uint32_t>(p);
      low[i] = bitcast<uint32_t>(half2_t{(half_t)rest(h[2 * i], (float)p[0]), (half_t)rest(h[2 * i + 1], (float)p[1])});
    } else {
      high[i] = pack_bf16x2(h[2 * i], h[2 * i + 1]);
      low[i] = pack_bf16x2(rest(h[2 * i], bitcast<float>(high[i] << 16)), rest(h[2 * i + 1], bitcast<float>(high[i] & 0xffff0000u)));
    }
  }
}

// 16 MT rows of a tile (which has `halves` times as many) x blocks of 64 outputs; RB blocks of 32 ranks.  Lane (m, q) has 16 neighbouring outputs of row m:
// tile j of the four 16-row tiles of B holds rows 16 (i / 4) + 4 j + i % 4 of the block.
template <typename T, typename TO, int MT, int RB>
__global__ __launch_bounds__(256) void low_rank_up_kernel(const UpArgs a) {
  typedef typename MmaOf<T>::type Mma;
  constexpr int W = 16 * sizeof(TO) / 16;  // 16-byte pieces of a lane's outputs
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
  const Tile<MT> tile(a.r, blockIdx.x, lane);
  const int slot0 = blockIdx.z * 16 * MT, live = tile.rows - slot0;
  if (live <= 0) return;
  const int frags = (live + 15) / 16 < MT ? (live + 15) / 16 : MT;
  int64_t row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) row[t] = tile.row(a.r, slot0 + t * 16 + r16);
  const bool with = tile.adapter != a.r.L;
  const float scaling = with ? a.scaling[tile.adapter] : 0.0f;
  const int blocks0 = (a.end0 + 63) / 64, blocks1 = blocks0 + (a.end1 - a.end0 + 63) / 64, blocks = blocks1 + (a.N - a.end1 + 63) / 64;
  int have = -1;  // the part of the outputs whose h is there
  uint4_t high[MT][RB], low[MT][RB];
  float back[MT];  // what the pieces' power of two takes back, times the scaling
  for (int i = 0; i < a.per_group; i += 4) {
    const int block = blockIdx.y * a.per_group + i + wave;
    if (block >= blocks) break;
    const int p = (block >= blocks0) + (block >= blocks1);
    const int n0 = p == 0 ? block * 64 : p == 1 ? a.end0 + (block - blocks0) * 64 : a.end1 + (block - blocks1) * 64;
    const int end = p == 0 ? a.end0 : p == 1 ? a.end1 : a.N;
    const int n = n0 + q * 16;
    const bool there = n < end;
    uint4_t y[MT][W];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t >= frags) break;
#pragma unroll
      for (int v = 0; v < W; ++v)
        if (there && slot0 + t * 16 + r16 < tile.rows) y[t][v] = __builtin_nontemporal_load((const uint4_t*)((const TO*)a.Y + row[t] * a.N + n) + v);
    }
    if (!with) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < W; ++v)
          if (there && slot0 + t * 16 + r16 < tile.rows) *((uint4_t*)((TO*)a.out + row[t] * a.N + n) + v) = y[t][v];
      continue;
    }
    uint4_t b[4][RB];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = n0 + 16 * (r16 >> 2) + 4 * j + (r16 & 3);
      const T* const w = (const T*)a.B + ((int64_t)tile.adapter * a.N + (at < end ? at : n0)) * a.rank + q * 8;
#pragma unroll
      for (int c = 0; c < RB; ++c) b[j][c] = c * 32 + q * 8 < a.rank ? *(const uint4_t*)(w + c * 32) : uint4_t{0, 0, 0, 0};
    }
    if (p != have) {
      have = p;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t >= frags) break;
        float h[RB][8];
#pragma unroll
        for (int c = 0; c < RB; ++c) {
#pragma unroll
          for (int k = 0; k < 8; ++k) h[c][k] = 0.0f;
          if (c * 32 + q * 8 < a.rank) {
            const float* s = a.sums + row[t] * a.rows + p * a.rank + c * 32 + q * 8;
            for (int part = 0; part < a.parts; ++part, s += (int64_t)a.r.M * a.rows) {
              const float4_t u = *(const float4_t*)s, v = *(const float4_t*)(s + 4);
#pragma unroll
              for (int k = 0; k < 4; ++k) h[c][k] += u[k], h[c][4 + k] += v[k];
            }
          }
        }
        back[t] = scaling;
        if constexpr (std::is_same<T, half_t>::value) {
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(h[c][k]));
          top = fmaxf(top, __shfl_xor(top, 16)), top = fmaxf(top, __shfl_xor(top, 32));
          // 2^e <= top < 2^(e + 1), e from -100 to 126 (less is 0 to float16 beside any weight; infinities and NaN stay what they are)
          int e = (int)(bitcast<uint32_t>(top) >> 23) - 127;
          e = e < -100 ? -100 : e > 126 ? 126 : e;
          const float down = bitcast<float>((uint32_t)(127 - e) << 23), up = bitcast<float>((uint32_t)(127 + e) << 23);
          back[t] *= up;
#pragma unroll
          for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) h[c][k] *= down;
        }
#pragma unroll
        for (int c = 0; c < RB; ++c) two_pieces<T>(h[c], high[t][c], low[t][c]);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t >= frags) break;
      float4_t acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[j] = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < RB; ++c) acc[j] = Mma::mma(b[j][c], low[t][c], acc[j]);
#pragma unroll
        for (int c = 0; c < RB; ++c) acc[j] = Mma::mma(b[j][c], high[t][c], acc[j]);
      }
      if (!there || slot0 + t * 16 + r16 >= tile.rows) continue;
      uint4_t* const o = (uint4_t*)((TO*)a.out + row[t] * a.N + n);
      if constexpr (sizeof(TO) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float4_t z = bitcast<float4_t>(y[t][j]);
#pragma unroll
          for (int k = 0; k < 4; ++k) z[k] = __builtin_fmaf(back[t], acc[j][k], z[k]);
          o[j] = bitcast<uint4_t>(z);
        }
      } else {
#pragma unroll
        for (int v = 0; v < W; ++v) {
          uint4_t z;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t two = y[t][v][k];
            float f[2];
            if constexpr (std::is_same<T, half_t>::value) f[0] = (float)bitcast<half2_t>(two)[0], f[1] = (float)bitcast<half2_t>(two)[1];
            else f[0] = bitcast<float>(two << 16), f[1] = bitcast<float>(two & 0xffff0000u);
            const float4_t& s = acc[2 * v + (k >> 1)];
            f[0] = __builtin_fmaf(back[t], s[2 * (k & 1)], f[0]), f[1] = __builtin_fmaf(back[t], s[2 * (k & 1) + 1], f[1]);
            if constexpr (std::is_same<T, half_t>::value) z[k] = bitcast<uint32_t>(half2_t{(half_t)f[0], (half_t)f[1]});
            else z[k] = pack_bf16x2(f[0], f[1]);
          }
          o[v] = z;
        }
      }
    }
  }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------
inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
inline int64_t most_tiles(int64_t M, int64_t L) { return M <= kInlineRows ? M : M / 64 + (L + 1 < M ? L + 1 : M); }
int64_t plan_bytes(int64_t M, int64_t L) { return M <= kInlineRows ? 0 : align256((tiles_at(M) + 4 * most_tiles(M, L)) * 4); }
int64_t most_parts(int64_t K) { return K >= 4096 ? 16 : (K + 255) / 256; }
// parts * M is at most this for more than one part
constexpr int64_t kPartRows = 32768;
int64_t parts_of(int64_t M, int64_t L, int64_t groups, int64_t K) {
  const int64_t tiles = most_tiles(M, L) * groups;
  int64_t parts = (512 + tiles - 1) / tiles;
  if (parts > most_parts(K)) parts = most_parts(K);
  if (parts * M > kPartRows) parts = kPartRows / M;
  return parts < 1 ? 1 : parts;
}

struct Call {
  Rows r;
  const void *X, *Y, *A, *B;
  const float* scaling;
  void* out;
  int32_t* plan;
  float* sums;
  int K, N, rank, rows, end0, end1;
};

template <typename T, int MT, int NT>
int run_down(const Call& c, int64_t tiles, int64_t* parts, hipStream_t st) {
  const int groups = (c.rows + 16 * NT - 1) / (16 * NT);
  int64_t want = parts_of(c.r.M, c.r.L, groups, c.K);
  const int part_k = (int)((ceil_div(c.K, want) + 255) / 256 * 256);
  *parts = ceil_div(c.K, part_k);
  const DownArgs a{c.r, c.X, c.A, c.sums, c.K, c.rows, part_k};
  low_rank_down_kernel<T, MT, NT><<<dim3((unsigned)tiles, (unsigned)*parts, (unsigned)groups), 256, 0, st>>>(a);
  return check_launch("tlq_low_rank_update", "low_rank_down_kernel") ? 0 : 1;
}

template <typename T, typename TO, int MT, int RB>
int run_up(const Call& c, int64_t tiles, int64_t parts, int tile_rows, hipStream_t st) {
  const int blocks = (c.end0 + 63) / 64 + (c.end1 - c.end0 + 63) / 64 + (c.N - c.end1 + 63) / 64;
  int per_group = 4;
  while (per_group < 64 && tiles * ceil_div(blocks, (int64_t)per_group) > 2048) per_group += 4;
  while (ceil_div(blocks, (int64_t)per_group) > 65535) per_group *= 2;
  const UpArgs a{c.r, c.Y, c.B, c.scaling, c.sums, c.out, c.N, c.rank, c.rows, (int)parts, c.end0, c.end1, per_group};
  low_rank_up_kernel<T, TO, MT, RB><<<dim3((unsigned)tiles, (unsigned)ceil_div(blocks, (int64_t)per_group), (unsigned)(tile_rows / (16 * MT))), 256, 0, st>>>(a);
  return check_launch("tlq_low_rank_update", "low_rank_up_kernel") ? 0 : 1;
}

template <typename T, typename TO>
int run_low_rank(Call c, hipStream_t st) {
  const int64_t tiles = most_tiles(c.r.M, c.r.L);
  int64_t parts = 1;
  if (c.r.M <= kInlineRows) {
    if (run_down<T, 1, 1>(c, tiles, &parts, st)) return 1;
    if (c.rank <= 32) return run_up<T, TO, 1, 1>(c, tiles, parts, 16, st);
    if (c.rank <= 64) return run_up<T, TO, 1, 2>(c, tiles, parts, 16, st);
    return run_up<T, TO, 1, 4>(c, tiles, parts, 16, st);
  }
  low_rank_plan_kernel<<<1, 1024, 0, st>>>(c.r.ids, c.plan, c.r.M, c.r.L);
  if (!check_launch("tlq_low_rank_update", "low_rank_plan_kernel")) return 1;
  c.r.plan = c.plan;
  if (c.rows <= 16 ? run_down<T, 4, 1>(c, tiles, &parts, st) : c.rows <= 32 ? run_down<T, 4, 2>(c, tiles, &parts, st) : run_down<T, 4, 4>(c, tiles, &parts, st)) return 1;
  if (c.rank <= 32) return run_up<T, TO, 4, 1>(c, tiles, parts, 64, st);
  if (c.rank <= 64) return run_up<T, TO, 2, 2>(c, tiles, parts, 64, st);
  return run_up<T, TO, 2, 4>(c, tiles, parts, 64, st);
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
  const int64_t few = most_parts(K) * M, many = M > kPartRows ? M : kPartRows;
  return plan_bytes(M, L) + (few < many ? few : many) * parts * rank * 4;
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
