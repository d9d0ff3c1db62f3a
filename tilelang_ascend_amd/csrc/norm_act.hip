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

// Any N: a work-group a row, one value per lane and step, the row read twice (with a residual the sum is read back from H by the lane that wrote it:
// H may be the residual itself).
template <typename T>
__global__ __launch_bounds__(256) void norm_any_kernel(const NormArgs a) {
  __shared__ float part[2][2][4];
  const int tid = threadIdx.x, N = a.N;
  int it = 0;
  for (int64_t m = blockIdx.x; m < a.M; m += a.blocks, it ^= 1) {
    const T *x = (const T*)a.X + m * N, *r = (const T*)a.R + m * N, *w = (const T*)a.W;
    T* const h = (T*)a.H + m * N;
    float ss = 0.0f, amax = 0.0f;
    for (int n = tid; n < N; n += 256) {
      float z = to_float(x[n]);
      if (a.R) {
        const T sum = from_float<T>(z + to_float(r[n]));
        h[n] = sum, z = to_float(sum);
      }
      ss += z * z;
      amax = fmaxf(amax, fabsf(z * to_float(w[n])));
    }
    ss = wave_sum(ss), amax = wave_max(amax);
    if ((tid & 63) == 0) part[it][0][tid >> 6] = ss, part[it][1][tid >> 6] = amax;
    __syncthreads();  // (part[] alternates: one barrier a row)
    ss = (part[it][0][0] + part[it][0][1]) + (part[it][0][2] + part[it][0][3]);
    amax = fmaxf(fmaxf(part[it][1][0], part[it][1][1]), fmaxf(part[it][1][2], part[it][1][3]));
    const float rstd = 1.0f / sqrtf(ss / (float)N + a.eps);
    const RowCodes c = row_codes(amax, rstd, a.round_scale);
    const float rcp = 1.0f / c.scale;
    if (a.S && tid == 0) a.S[m] = c.scale;
    const T* const from = a.R ? h : x;
    for (int n = tid; n < N; n += 256) {
      const float v = to_float(from[n]) * to_float(w[n]), y = v * rstd;
      if (a.Q) {
        const float t = v * c.mul;
        a.Q[m * N + n] = (int8_t)(c.mul == 0.0f ? quant1(y, c.scale, rcp) : code_near(t) ? (uint32_t)code_exact(v, t, amax) : quant1(t, 1.0f, 1.0f));
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

// Any N: a work-group a row, one value per lane and step; codes are made of a second look at the row.
template <typename T>
__global__ __launch_bounds__(256) void gated_any_kernel(const GatedArgs a) {
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
    if (!a.Q) continue;
    amax = wave_max(amax);
    if ((tid & 63) == 0) part[it][tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part[it][0], part[it][1]), fmaxf(part[it][2], part[it][3]));
    const float scale = row_scale(amax, a.round_scale), rcp = 1.0f / scale;
    if (tid == 0) a.S[m] = scale;
    for (int n = tid; n < N; n += 256) a.Q[m * N + n] = (int8_t)quant1(value(n), scale, rcp);
  }
}

int grid_of(int64_t M) {  // rows walk over a resident grid
  int cus = tlq_device_cu_count();
  if (cus <= 0) cus = 256;
  return (int)(M < (int64_t)cus * 8 ? M : (int64_t)cus * 8);
}

template <typename T>
int run_norm(NormArgs a, hipStream_t st) {
  a.blocks = grid_of(a.M);
  norm_any_kernel<T><<<a.blocks, 256, 0, st>>>(a);
  return check_launch("tlq_residual_rms_norm", "norm_any_kernel") ? 0 : 1;
}

template <typename T>
int run_gated(GatedArgs a, hipStream_t st) {
  a.blocks = grid_of(a.M);
  gated_any_kernel<T><<<a.blocks, 256, 0, st>>>(a);
  return check_launch("tlq_gated_silu", "gated_any_kernel") ? 0 : 1;
}

// What both entry points ask of their sizes and outputs.
int check_rows(const char* what, int64_t M, int64_t N, int dtype) {
  TLQ_REQUIRE(M >= 0 && M < ((int64_t)1 << 40) && N >= 1 && N < ((int64_t)1 << 30), "%s: bad shape M=%lld N=%lld", what, (long long)M, (long long)N);
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
