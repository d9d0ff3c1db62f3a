// What stands between two products of a transformer block: the residual's addition with the root-mean-square norm, and the gated activation
// of an MLP; outputs in the activations' type and / or in the codes and scales of the int8 products.
//   norm:   h = T(x + residual) (h = x without one), v = h * w, y = v * rstd, rstd = 1 / sqrt(mean(h^2) + eps)
//   gated:  y = silu(x[:N]) * x[N:]
//   Y = T(y);  S = max(max |y|, 1e-4) / 127 (round_scale: the next power of two);  Q = rint(clamp(y / S, -127, 127)), half to even
// y is fp32 and rounded once, into either output: the codes are those of y, not of Y.
//
// h and w are 16-bit, so v is exact in fp32 (22 bits at most), and rstd cancels out of the codes of a norm where S is not the floor:
// Q = rint(127 v / max |v|), which is decided exactly (code_of): the codes do not depend on how the sum of squares was formed.
#include "row_quant.h"
#include "silu.h"

namespace tlq {
namespace {

// The code of v: v over unit = amax / 127, from t = v * (127 / amax), which is at most 127 * 2^-23 off.  Nearer to the middle of two codes than
// that the whole numbers decide: 254 |v| against (2 k + 1) amax in binary64, which holds both (22 bits and 8), halves to the even code.
__device__ __forceinline__ bool code_near(float t) {
  const float n = (t + 12582912.0f) - 12582912.0f;
  return fabsf(t - n) > 0.5f - 0x1p-15f;
}
__device__ __forceinline__ int code_exact(float v, float t, float amax) {
  const float k = floorf(fabsf(t));
  const double middle = (double)(2.0f * k + 1.0f) * (double)amax, twice = 254.0 * (double)fabsf(v);
  const int n = (int)k + (twice > middle || (twice == middle && ((int)k & 1)) ? 1 : 0);
  return v < 0.0f ? -n : n;
}

// What quant1 divides by in a row of this scale.  A row with an infinity has an infinite scale, whose reciprocal is 0: over 0 its finite values get code 0, and
// the infinity, as NaN does, -127.
__device__ __forceinline__ float divisor(float scale) { return scale < __builtin_inff() ? scale : 0.0f; }

struct NormArgs {
  const void *X, *R, *W;  // R: null without a residual
  void *H, *Y;            // H: null without a residual; Y, or Q and S: null if not wanted
  int8_t* Q;
  float* S;
  int64_t M;
  int N, round_scale, blocks;
  float eps;
};

// What a row's codes are made with.
struct RowCodes {
  float scale, amax, mul;  // y / scale; v * (127 / amax) where rstd cancels (mul: that; 0: it does not)
};
__device__ __forceinline__ RowCodes row_codes(float amax_v, float rstd, int round_scale) {
  const float amax = amax_v * rstd;
  RowCodes c;
  c.scale = row_scale(amax, round_scale);  // (a maximum of NaN is the floor's)
  c.amax = amax_v;
  c.mul = !round_scale && amax >= 1e-4f && amax < __builtin_inff() ? 127.0f / amax_v : 0.0f;
  return c;
}

__device__ __forceinline__ float wave_sum(float v) {
  auto dpp = [&](auto ctrl) { v += bitcast<float>(__builtin_amdgcn_update_dpp(0, bitcast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false)); };
  dpp(std::integral_constant<int, 0xb1>{}), dpp(std::integral_constant<int, 0x4e>{}), dpp(std::integral_constant<int, 0x141>{}), dpp(std::integral_constant<int, 0x140>{});
  const auto rows = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
  v = bitcast<float>((uint32_t)rows[0]) + bitcast<float>((uint32_t)rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
  return bitcast<float>((uint32_t)halves[0]) + bitcast<float>((uint32_t)halves[1]);
}

// Eight neighbouring values of a row, as they lie in memory.
template <typename T>
__device__ __forceinline__ float value_of(const uint4_t& w, int i) {
  if constexpr (std::is_same<T, half_t>::value) return (float)bitcast<half8_t>(w)[i];
  else return bitcast<float>((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, half_t>::value) return bitcast<uint32_t>(half2_t{(half_t)lo, (half_t)hi});
  else return pack_bf16x2(lo, hi);
}
template <typename T>
__device__ __forceinline__ uint4_t pack8(const float (&f)[8]) {
  return uint4_t{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])};
}
__device__ __forceinline__ uint2_t pack_codes(const uint32_t (&c)[8]) {
  uint2_t o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * h + 1], c[4 * h], 0x0c0c0400u);
    o[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * h + 3], c[4 * h + 2], 0x0c0c0400u), lo, 0x05040100u);
  }
  return o;
}

// Eight values from p on, `left` of them in the row.  ANY: rows of any length that begin anywhere -- the memory takes accesses of 16 bytes at any
// address (3000 x 4099 bf16, both outputs: 68 us a value at a time) --, otherwise all eight are there and p is 16-byte aligned.  ONCE: nobody reads them again (non-temporal loads of the
// rows: 8192 x 8192 bf16 with a residual 90.8 us, 93.1 with ordinary ones, gated 8192 x 14336 with codes 102 / 110; of the weights too 119).
template <bool ANY, bool ONCE = true, typename T>
__device__ __forceinline__ uint4_t load8(const T* p, int left) {
  if constexpr (!ANY) {
    return ONCE ? __builtin_nontemporal_load((const uint4_t*)p) : *(const uint4_t*)p;
  } else {
    struct __attribute__((packed, aligned(2))) Packed { uint4_t v; };
    if (left >= 8) return ((const Packed*)p)->v;
    uint4_t o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < left) o[i >> 1] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i & 1));
    return o;
  }
}
template <bool ANY, typename T>
__device__ __forceinline__ void store8(T* p, const uint4_t& v, int left) {
  if constexpr (!ANY) {
    *(uint4_t*)p = v;
  } else {
    struct __attribute__((packed, aligned(2))) Packed { uint4_t v; };
    if (left >= 8) {
      ((Packed*)p)->v = v;
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < left) ((uint16_t*)p)[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
    }
  }
}
template <bool ANY>
__device__ __forceinline__ void store_codes(int8_t* p, const uint2_t& v, int left) {
  if constexpr (!ANY) {
    *(uint2_t*)p = v;
  } else {
    struct __attribute__((packed, aligned(1))) Packed { uint2_t v; };
    if (left >= 8) {
      ((Packed*)p)->v = v;
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < left) p[i] = (int8_t)(v[i >> 2] >> (8 * (i & 3)));
    }
  }
}

// Up to 32768 values: WPR wavefronts of a work-group share a row, a lane keeps CH chunks of 8 values of it and of the weights, the row is read
// once.  One barrier a row: the sum of squares and max |v| are formed together, since v does not wait for rstd.
template <typename T, int CH, int WPR, int THREADS, bool ANY>
__global__ __launch_bounds__(THREADS) void norm_rows_kernel(const NormArgs a) {
  constexpr int ROWS = THREADS / 64 / WPR, LANES = 64 * WPR;
  __shared__ float part[2][2][THREADS / 64];
  const int wave = threadIdx.x >> 6, first = (wave / WPR) * WPR, at = threadIdx.x - first * 64, chunks = (a.N + 7) >> 3;
  const float inv_n = 1.0f / (float)a.N;
  uint4_t w[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * LANES + at;
    w[c] = i < chunks ? load8<ANY, false>((const T*)a.W + i * 8, a.N - i * 8) : uint4_t{0, 0, 0, 0};
  }
  int it = 0;
  for (int64_t m0 = (int64_t)blockIdx.x * ROWS; m0 < a.M; m0 += (int64_t)a.blocks * ROWS, it ^= 1) {
    const int64_t own = m0 + wave / WPR, m = own < a.M ? own : a.M - 1;  // (a wavefront without a row goes through the last one's and writes nothing)
    const bool live = own < a.M;
    const int64_t row = m * a.N;
    uint4_t h[CH];
    float ss = 0.0f, amax = 0.0f;
    uint4_t r[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at;
      const int from = (i < chunks ? i : chunks - 1) * 8;  // (a lane without a chunk reads the last one)
      h[c] = load8<ANY>((const T*)a.X + row + from, a.N - from);
      if (a.R) r[c] = load8<ANY>((const T*)a.R + row + from, a.N - from);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at;
      if (a.R) {
        float sum[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = value_of<T>(h[c], k) + value_of<T>(r[c], k);
        h[c] = pack8<T>(sum);
        if (live && i < chunks) store8<ANY>((T*)a.H + row + i * 8, h[c], a.N - i * 8);
      }
      if (i >= chunks) h[c] = uint4_t{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float z = value_of<T>(h[c], k);
        ss = __builtin_fmaf(z, z, ss);
        amax = fmaxf(amax, fabsf(z * value_of<T>(w[c], k)));
      }
    }
    ss = wave_sum(ss);
    if (a.Q) amax = wave_max(amax);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) part[it][0][wave] = ss, part[it][1][wave] = amax;
      __syncthreads();  // (part[] alternates between rows)
      ss = 0.0f;
#pragma unroll
      for (int k = 0; k < WPR; ++k) ss += part[it][0][first + k], amax = fmaxf(amax, part[it][1][first + k]);
    }
    const float rstd = 1.0f / sqrtf(ss * inv_n + a.eps);
    if (a.Y && live) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int i = c * LANES + at;
        if (i >= chunks) break;
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = value_of<T>(h[c], k) * value_of<T>(w[c], k) * rstd;
        store8<ANY>((T*)a.Y + row + i * 8, pack8<T>(y), a.N - i * 8);
      }
    }
    if (!a.Q) continue;
    const RowCodes codes = row_codes(amax, rstd, a.round_scale);
    if (live && at == 0) a.S[m] = codes.scale;
    if (!live) continue;
    const float rcp = 1.0f / codes.scale, over = divisor(codes.scale);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at;
      if (i >= chunks) break;
      uint32_t q[8];
      if (codes.mul != 0.0f) {
        bool near = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = value_of<T>(h[c], k) * value_of<T>(w[c], k) * codes.mul;
          q[k] = quant1(t, 1.0f, 1.0f);
          near |= code_near(t);
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(near) != 0, 0)) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float v = value_of<T>(h[c], k) * value_of<T>(w[c], k), t = v * codes.mul;
            if (code_near(t)) q[k] = (uint32_t)code_exact(v, t, amax);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = quant1(value_of<T>(h[c], k) * value_of<T>(w[c], k) * rstd, over, rcp);
      }
      store_codes<ANY>(a.Q + row + i * 8, pack_codes(q), a.N - i * 8);
    }
  }
}

// Longer rows: a work-group a row, one value per lane and step, the row read twice (with a residual the sum is read back from H by the lane that wrote
// it: H may be the residual itself).  A lane has up to 2^22 squares: sums of kRun of them in fp32, those in binary64 (one sum in fp32 was 0.3 % off for equal values
// in rows of 2^26, and 3 % in the longest).  Bounded by the latency of two-byte loads and by the second reading: rows of 53248 bf16 with a residual, us, 16 bits / codes:
// 1 97 / 109, 64 142 / 148, 2000 486 / 470 (852 and 745 MB: 1.8 and 1.6 TB/s).
constexpr int kRun = 64;
template <typename T>
__global__ __launch_bounds__(256) void norm_long_kernel(const NormArgs a) {
  __shared__ float part[2][2][4];
  const int tid = threadIdx.x, N = a.N;
  int it = 0;
  for (int64_t m = blockIdx.x; m < a.M; m += a.blocks, it ^= 1) {
    const T *x = (const T*)a.X + m * N, *r = (const T*)a.R + m * N, *w = (const T*)a.W;
    T* const h = (T*)a.H + m * N;
    float amax = 0.0f;
    double all = 0.0;
    for (int n0 = tid; n0 < N; n0 += kRun * 256) {
      float run = 0.0f;
      for (int n = n0; n < N && n < n0 + kRun * 256; n += 256) {
        float z = to_float(x[n]);
        if (a.R) {
          const T sum = from_float<T>(z + to_float(r[n]));
          h[n] = sum, z = to_float(sum);
        }
        run += z * z;
        amax = fmaxf(amax, fabsf(z * to_float(w[n])));
      }
      all += (double)run;
    }
    float ss = wave_sum((float)all);
    amax = wave_max(amax);
    if ((tid & 63) == 0) part[it][0][tid >> 6] = ss, part[it][1][tid >> 6] = amax;
    __syncthreads();  // (part[] alternates: one barrier a row)
    ss = (part[it][0][0] + part[it][0][1]) + (part[it][0][2] + part[it][0][3]);
    amax = fmaxf(fmaxf(part[it][1][0], part[it][1][1]), fmaxf(part[it][1][2], part[it][1][3]));
    const float rstd = 1.0f / sqrtf(ss / (float)N + a.eps);
    const RowCodes c = row_codes(amax, rstd, a.round_scale);
    const float rcp = 1.0f / c.scale, over = divisor(c.scale);
    if (a.S && tid == 0) a.S[m] = c.scale;
    const T* const from = a.R ? h : x;
    for (int n = tid; n < N; n += 256) {
      const float v = to_float(from[n]) * to_float(w[n]), y = v * rstd;
      if (a.Q) {
        const float t = v * c.mul;
        a.Q[m * N + n] = (int8_t)(c.mul == 0.0f ? quant1(y, over, rcp) : code_near(t) ? (uint32_t)code_exact(v, t, amax) : quant1(t, 1.0f, 1.0f));
      }
      if (a.Y) ((T*)a.Y)[m * N + n] = from_float<T>(y);
    }
  }
}

struct GatedArgs {
  const void* X;
  void* Y;
  int8_t* Q;
  float* S;
  int64_t M;
  int N, round_scale, blocks;
};

// Eight outputs of eight gates and eight ups.
template <typename T>
__device__ __forceinline__ void gated8(const uint4_t& g, const uint4_t& u, float (&y)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float4_t a, b;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = value_of<T>(g, 4 * h + k), b[k] = value_of<T>(u, 4 * h + k);
    const float4_t z = silu_times(a, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) y[4 * h + k] = z[k];
  }
}

// Y alone: a lane per chunk of 8 values.  A work-group has 256 chunks of a row (segs of them make a row), or several short rows.
template <typename T, bool ANY>
__global__ __launch_bounds__(256) void gated_flat_kernel(const GatedArgs a, int segs, int rows) {
  const int chunks = (a.N + 7) >> 3, group = blockIdx.x / segs, seg = blockIdx.x - group * segs;
  int of_row = threadIdx.x, chunk = seg * 256 + threadIdx.x;
  int64_t m = group;
  if (rows > 1) {
    of_row = threadIdx.x / chunks, chunk = threadIdx.x - of_row * chunks, m = (int64_t)group * rows + of_row;
    if (of_row >= rows) return;
  }
  if (m >= a.M || chunk >= chunks) return;
  const T* const x = (const T*)a.X + m * 2 * a.N + chunk * 8;
  const int left = a.N - chunk * 8;
  const uint4_t g = load8<ANY>(x, left), u = load8<ANY>(x + a.N, left);
  float y[8];
  gated8<T>(g, u, y);
  store8<ANY>((T*)a.Y + m * a.N + chunk * 8, pack8<T>(y), left);
}

// With codes, up to 32768 values: WPR wavefronts of a work-group share a row, whose values stay in registers between the maximum and the codes.
template <typename T, int CH, int WPR, int THREADS, bool ANY>
__global__ __launch_bounds__(THREADS) void gated_rows_kernel(const GatedArgs a) {
  constexpr int ROWS = THREADS / 64 / WPR, LANES = 64 * WPR;
  __shared__ float part[2][THREADS / 64];
  const int wave = threadIdx.x >> 6, first = (wave / WPR) * WPR, at = threadIdx.x - first * 64, chunks = (a.N + 7) >> 3;
  int it = 0;
  for (int64_t m0 = (int64_t)blockIdx.x * ROWS; m0 < a.M; m0 += (int64_t)a.blocks * ROWS, it ^= 1) {
    const int64_t own = m0 + wave / WPR, m = own < a.M ? own : a.M - 1;  // (a wavefront without a row goes through the last one's and writes nothing)
    const bool live = own < a.M;
    const T* const x = (const T*)a.X + m * 2 * a.N;
    uint4_t g[CH], u[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at, from = (i < chunks ? i : chunks - 1) * 8;  // (a lane without a chunk reads the last one: the maximum stays what it is)
      g[c] = load8<ANY>(x + from, a.N - from), u[c] = load8<ANY>(x + a.N + from, a.N - from);
    }
    float y[CH][8], amax = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at;
      gated8<T>(g[c], u[c], y[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(y[c][k]));
      if (a.Y && live && i < chunks) store8<ANY>((T*)a.Y + m * a.N + i * 8, pack8<T>(y[c]), a.N - i * 8);
    }
    amax = wave_max(amax);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) part[it][wave] = amax;
      __syncthreads();  // (part[] alternates between rows)
#pragma unroll
      for (int k = 0; k < WPR; ++k) amax = fmaxf(amax, part[it][first + k]);
    }
    const float scale = row_scale(amax, a.round_scale), rcp = 1.0f / scale, over = divisor(scale);
    if (!live) continue;
    if (at == 0) a.S[m] = scale;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * LANES + at;
      if (i >= chunks) break;
      uint32_t q[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = quant1(y[c][k], over, rcp);
      store_codes<ANY>(a.Q + m * a.N + i * 8, pack_codes(q), a.N - i * 8);
    }
  }
}

// Longer rows with codes: a work-group a row, one value per lane and step; codes are made of a second look at the row.  (Rows of 53248 bf16: 1 78 us, 64 118, 2000 296 for 533 MB.)
template <typename T>
__global__ __launch_bounds__(256) void gated_long_kernel(const GatedArgs a) {
  __shared__ float part[2][4];
  const int tid = threadIdx.x, N = a.N;
  int it = 0;
  for (int64_t m = blockIdx.x; m < a.M; m += a.blocks, it ^= 1) {
    const T* const x = (const T*)a.X + m * 2 * N;
    const auto value = [&](int n) __attribute__((always_inline)) {
      const float4_t g = {to_float(x[n]), 0.0f, 0.0f, 0.0f}, u = {to_float(x[N + n]), 0.0f, 0.0f, 0.0f};
      return silu_times(g, u)[0];
    };
    float amax = 0.0f;
    for (int n = tid; n < N; n += 256) {
      const float y = value(n);
      if (a.Y) ((T*)a.Y)[m * N + n] = from_float<T>(y);
      amax = fmaxf(amax, fabsf(y));
    }
    amax = wave_max(amax);
    if ((tid & 63) == 0) part[it][tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part[it][0], part[it][1]), fmaxf(part[it][2], part[it][3]));
    const float scale = row_scale(amax, a.round_scale), rcp = 1.0f / scale, over = divisor(scale);
    if (tid == 0) a.S[m] = scale;
    for (int n = tid; n < N; n += 256) a.Q[m * N + n] = (int8_t)quant1(value(n), over, rcp);
  }
}

constexpr int kLongRow = 32768;
constexpr int64_t kMostGroups = ((int64_t)1 << 24) - 1;  // work-groups of 256 threads of a launch, which has fewer than 2^32 threads

// Work-groups for this many rows (or groups of rows): up to 64 a CU, which then walk on.  8192 x 8192 bf16 with a residual: 90.7 us, 94.8 with 8 a CU,
// 94 with 4; on rows of 1024 to 4096 values level.
int grid_of(int64_t groups) {
  int cus = tlq_device_cu_count();
  if (cus <= 0) cus = 256;
  return (int)(groups < (int64_t)cus * 64 ? groups : (int64_t)cus * 64);
}

inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

template <typename T>
int run_norm(NormArgs a, hipStream_t st) {
  if (a.N <= kLongRow) {
    const bool any = !(a.N % 8 == 0 && aligned(a.X, 16) && aligned(a.R, 16) && aligned(a.W, 16) && aligned(a.H, 16) && aligned(a.Y, 16) && aligned(a.Q, 8));
#define TLQ_NORM(CH, WPR, THREADS)                                                            \
  do {                                                                                        \
    a.blocks = grid_of(ceil_div(a.M, (int64_t)(THREADS / 64 / WPR)));                         \
    if (any) norm_rows_kernel<T, CH, WPR, THREADS, true><<<a.blocks, THREADS, 0, st>>>(a);    \
    else norm_rows_kernel<T, CH, WPR, THREADS, false><<<a.blocks, THREADS, 0, st>>>(a);       \
  } while (0)
    // the fewest chunks a lane with up to eight wavefronts a row (us, bf16 with a residual; four wavefronts / eight / sixteen: 1 x 4096 2.7 / 2.45 / 2.6,
    // 512 x 4096 4.85 / 4.7 / 5.5, 4099 x 4096 27.8 / 26.5 / -, 2048 x 4096 14.8 / 13.9 / 16.5, 8192 x 8192 92.5 / 90.7 / 91.9, 4096 x 16384 109.3 / 109.3 / 112.4;
    // one / four: 4096 x 1024 8.2 / 8.6, 1024 x 1024 3.97 / 4.05, 4096 x 2048 13.1 / 13.5, 1021 x 2048 4.8 / 4.4)
    if (a.N <= 512) TLQ_NORM(1, 1, 256);
    else if (a.N <= 1024) TLQ_NORM(2, 1, 256);
    else if (a.N <= 2048) TLQ_NORM(1, 4, 256);
    else if (a.N <= 4096) TLQ_NORM(1, 8, 512);
    else if (a.N <= 8192) TLQ_NORM(2, 8, 512);
    else if (a.N <= 16384) TLQ_NORM(4, 8, 512);
    else TLQ_NORM(4, 16, 1024);
#undef TLQ_NORM
    return check_launch("tlq_residual_rms_norm", "norm_rows_kernel") ? 0 : 1;
  }
  a.blocks = grid_of(a.M);
  norm_long_kernel<T><<<a.blocks, 256, 0, st>>>(a);
  return check_launch("tlq_residual_rms_norm", "norm_long_kernel") ? 0 : 1;
}

template <typename T>
int run_gated(GatedArgs a, hipStream_t st) {
  const char* const what = "tlq_gated_silu";
  const bool any = !(a.N % 8 == 0 && aligned(a.X, 16) && aligned(a.Y, 16) && aligned(a.Q, 8));
  if (!a.Q) {
    const int chunks = (a.N + 7) / 8, segs = (chunks + 255) / 256, rows = chunks > 128 ? 1 : 256 / chunks;
    const int64_t most = kMostGroups / segs * rows;  // rows of a launch
    for (int64_t m = 0; m < a.M; m += most) {
      GatedArgs part = a;
      part.X = (const T*)a.X + m * 2 * a.N, part.Y = (T*)a.Y + m * a.N, part.M = a.M - m < most ? a.M - m : most;
      const unsigned blocks = (unsigned)(ceil_div(part.M, (int64_t)rows) * segs);
      if (any) gated_flat_kernel<T, true><<<blocks, 256, 0, st>>>(part, segs, rows);
      else gated_flat_kernel<T, false><<<blocks, 256, 0, st>>>(part, segs, rows);
      if (!check_launch(what, "gated_flat_kernel")) return 1;
    }
    return 0;
  }
  if (a.N > kLongRow) {
    a.blocks = grid_of(a.M);
    gated_long_kernel<T><<<a.blocks, 256, 0, st>>>(a);
    return check_launch(what, "gated_long_kernel") ? 0 : 1;
  }
#define TLQ_GATED(CH, WPR, THREADS)                                                          \
  do {                                                                                       \
    a.blocks = grid_of(ceil_div(a.M, (int64_t)(THREADS / 64 / WPR)));                        \
    if (any) gated_rows_kernel<T, CH, WPR, THREADS, true><<<a.blocks, THREADS, 0, st>>>(a);  \
    else gated_rows_kernel<T, CH, WPR, THREADS, false><<<a.blocks, THREADS, 0, st>>>(a);     \
  } while (0)
  // the norm's table: codes alone, bf16, us, fewer wavefronts a row (four to 8192 values) / this / more (eight to 4096, sixteen to 16384): 67 x 14336 4.3 / 4.3 / 4.4, 2048 x 14336
  // 25.7 / 25.8 / 27.5, 512 x 11008 7.1 / 7.2 / 7.4, 512 x 8192 5.6 / 5.4 / 5.5, 4096 x 8192 28.0 / 27.7 / 31.2, 1024 x 4096 5.4 / 5.6 / 5.6, 4096 x 2048 9.1 / 9.1 / 12.9, 4096 x 1024
  // 7.5 / 5.3 / 11.5; four are faster where many rows have up to 4096 values (8192 x 4096 27.3 / 30.2 / 30.5)
  if (a.N <= 512) TLQ_GATED(1, 1, 256);
  else if (a.N <= 1024) TLQ_GATED(2, 1, 256);
  else if (a.N <= 2048) TLQ_GATED(1, 4, 256);
  else if (a.N <= 4096) TLQ_GATED(1, 8, 512);
  else if (a.N <= 8192) TLQ_GATED(2, 8, 512);
  else if (a.N <= 16384) TLQ_GATED(4, 8, 512);
  else TLQ_GATED(4, 16, 1024);
#undef TLQ_GATED
  return check_launch(what, "gated_rows_kernel") ? 0 : 1;
}

// What both entry points ask of their sizes and outputs.
int check_rows(const char* what, int64_t M, int64_t N, int dtype) {
  TLQ_REQUIRE(M >= 0 && M < ((int64_t)1 << 31) && N >= 1 && N < ((int64_t)1 << 30), "%s: bad shape M=%lld N=%lld", what, (long long)M, (long long)N);
  TLQ_REQUIRE(dtype == TLQ_F16 || dtype == TLQ_BF16, "%s: dtype must be float16 or bfloat16 (got %d)", what, dtype);
  return 0;
}
int check_outputs(const char* what, const void* Y, const void* Q, const void* S) {
  TLQ_REQUIRE(Y || Q, "%s: an output is wanted: Y, or Q and S", what);
  TLQ_REQUIRE(!Q == !S, "%s: Q and S are wanted together", what);
  TLQ_REQUIRE(((uintptr_t)Y & 1) == 0 && ((uintptr_t)S & 3) == 0, "%s: misaligned pointer", what);
  return 0;
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int tlq_residual_rms_norm(const void* X, const void* residual, const void* weight, void* H, void* Y, void* Q, void* S, int64_t M,
                                     int64_t N, float eps, int dtype, int round_scale, void* stream) {
  const char* const what = "tlq_residual_rms_norm";
  if (check_rows(what, M, N, dtype)) return 1;
  TLQ_REQUIRE(eps >= 1e-12f && eps <= 1.0f, "%s: eps must be between 1e-12 and 1 (got %g)", what, (double)eps);
  if (M == 0) return 0;
  TLQ_REQUIRE(X && weight, "%s: null pointer", what);
  TLQ_REQUIRE(!residual == !H, "%s: a residual and H are wanted together", what);
  TLQ_REQUIRE((((uintptr_t)X | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)H) & 1) == 0, "%s: misaligned pointer", what);
  if (check_outputs(what, Y, Q, S)) return 1;
  TLQ_REQUIRE(!H || H != Y, "%s: H and Y are two outputs (X's place is for one of them)", what);
  const NormArgs a{X, residual, weight, H, Y, (int8_t*)Q, (float*)S, M, (int)N, round_scale != 0, 0, eps};
  return dtype == TLQ_F16 ? run_norm<half_t>(a, (hipStream_t)stream) : run_norm<bf16_t>(a, (hipStream_t)stream);
}

extern "C" int tlq_gated_silu(const void* X, void* Y, void* Q, void* S, int64_t M, int64_t N, int dtype, int round_scale, void* stream) {
  const char* const what = "tlq_gated_silu";
  if (check_rows(what, M, N, dtype)) return 1;
  if (M == 0) return 0;
  TLQ_REQUIRE(X && ((uintptr_t)X & 1) == 0, "%s: null or misaligned pointer", what);
  if (check_outputs(what, Y, Q, S)) return 1;
  const GatedArgs a{X, Y, (int8_t*)Q, (float*)S, M, (int)N, round_scale != 0, 0};
  return dtype == TLQ_F16 ? run_gated<half_t>(a, (hipStream_t)stream) : run_gated<bf16_t>(a, (hipStream_t)stream);
}
