// Low-rank adapters of many requests beside a projection of up to three parts side by side (queries, keys, values; gate and up):
//   out[m, n] = rn(Y[m, n] + scaling[l] * sum_j h[m, p r + j] * B[l, n, j]),  h[m, i] = sum_k X[m, k] * A[l, i, k]
// l = ids[m], p the part that n lies in, r the rank; a row whose id names no adapter is out = Y.  h and the sums are fp32, rounded once, at the end.
#include "tlq_common.h"

namespace tlq {
namespace {

template <typename T>
__device__ __forceinline__ float widen(T v) { return to_float(v); }
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T narrow(float v) { return from_float<T>(v); }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }

struct LowRankArgs {
  const void *X, *Y;
  const int32_t* ids;
  const void *A, *B;
  const float* scaling;
  void* out;
  float* h;
  int M, L, rank, K, N, rows;  // rows: of an adapter's A, parts * rank
  int end0, end1;              // where the first and the second part end
};

// h: a wavefront per value.
template <typename T>
__global__ __launch_bounds__(256) void low_rank_down_kernel(const LowRankArgs a, int per_row) {
  const int lane = threadIdx.x & 63, m = blockIdx.x / per_row, i = (blockIdx.x - m * per_row) * 4 + (threadIdx.x >> 6), l = a.ids[m];
  if ((uint32_t)l >= (uint32_t)a.L || i >= a.rows) return;
  const T *x = (const T*)a.X + (int64_t)m * a.K, *w = (const T*)a.A + ((int64_t)l * a.rows + i) * a.K;
  float sum = 0.0f;
  for (int k = lane; k < a.K; k += 64) sum += to_float(x[k]) * to_float(w[k]);
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) a.h[(int64_t)m * a.rows + i] = sum;
}

// out: a lane per value.
template <typename T, typename TO>
__global__ __launch_bounds__(256) void low_rank_up_kernel(const LowRankArgs a, int per_row) {
  const int m = blockIdx.x / per_row, n = (blockIdx.x - m * per_row) * 256 + threadIdx.x, l = a.ids[m];
  if (n >= a.N) return;
  const int64_t at = (int64_t)m * a.N + n;
  float y = widen(((const TO*)a.Y)[at]);
  if ((uint32_t)l < (uint32_t)a.L) {
    const float* const h = a.h + (int64_t)m * a.rows + ((n >= a.end0) + (n >= a.end1)) * a.rank;
    const T* const w = (const T*)a.B + ((int64_t)l * a.N + n) * a.rank;
    float sum = 0.0f;
    for (int j = 0; j < a.rank; ++j) sum += h[j] * to_float(w[j]);
    y += a.scaling[l] * sum;
  }
  ((TO*)a.out)[at] = narrow<TO>(y);
}

template <typename T, typename TO>
int run_low_rank(const LowRankArgs& a, hipStream_t st) {
  const int per_down = (a.rows + 3) / 4, per_up = (a.N + 255) / 256;
  low_rank_down_kernel<T><<<a.M * per_down, 256, 0, st>>>(a, per_down);
  if (!check_launch("tlq_low_rank_update", "low_rank_down_kernel")) return 1;
  low_rank_up_kernel<T, TO><<<a.M * per_up, 256, 0, st>>>(a, per_up);
  return check_launch("tlq_low_rank_update", "low_rank_up_kernel") ? 0 : 1;
}

bool sizes_taken(int64_t M, int64_t L, int64_t rank, int64_t parts, int64_t K) {
  return M >= 0 && M < ((int64_t)1 << 24) && L >= 1 && L <= 4096 && (rank == 8 || rank == 16 || rank == 32 || rank == 64 || rank == 128) && parts >= 1 && parts <= 3 &&
         K >= 32 && K % 32 == 0 && K < ((int64_t)1 << 24);
}

}  // namespace
}  // namespace tlq

using namespace tlq;

extern "C" int64_t tlq_low_rank_update_workspace_bytes(int64_t M, int64_t L, int64_t rank, int64_t parts, int64_t K) {
  if (!sizes_taken(M, L, rank, parts, K)) return 0;
  return M * parts * rank * 4;
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
  TLQ_REQUIRE(M * ((N + 255) / 256) < ((int64_t)1 << 24) && M * parts * rank / 4 < ((int64_t)1 << 24), "%s: M=%lld rows of %lld values are too many for one call", what,
              (long long)M, (long long)N);
  TLQ_REQUIRE(X && Y && ids && A && B && scaling && out, "%s: null pointer", what);
  TLQ_REQUIRE((((uintptr_t)X | (uintptr_t)Y | (uintptr_t)A | (uintptr_t)B | (uintptr_t)out) & 15) == 0 && (((uintptr_t)ids | (uintptr_t)scaling) & 3) == 0,
              "%s: X, Y, A, B and out must be 16-byte aligned, ids and scaling to their type", what);
  const int64_t want = tlq_low_rank_update_workspace_bytes(M, L, rank, parts, K);
  TLQ_REQUIRE(workspace && workspace_bytes >= want && ((uintptr_t)workspace & 15) == 0, "%s: a 16-byte aligned workspace of %lld bytes is wanted (got %lld)", what,
              (long long)want, (long long)(workspace ? workspace_bytes : 0));
  const LowRankArgs a{X, Y, (const int32_t*)ids, A, B, (const float*)scaling, out, (float*)workspace, (int)M, (int)L, (int)rank, (int)K, (int)N,
                      (int)(parts * rank), (int)n0, (int)(n0 + n1)};
  hipStream_t st = (hipStream_t)stream;
  if (in_dtype == TLQ_F16) return out_dtype == TLQ_F32 ? run_low_rank<half_t, float>(a, st) : run_low_rank<half_t, half_t>(a, st);
  return out_dtype == TLQ_F32 ? run_low_rank<bf16_t, float>(a, st) : run_low_rank<bf16_t, bf16_t>(a, st);
}
