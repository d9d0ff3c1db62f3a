// W4A16 for large M, 256 activation rows per work-group: the panel kernel's structure (gemm_w4a16_panel.hip: packed weights
// copied global -> LDS as they are, dequantised on the MFMA operand read, step loop software-pipelined inside the
// wavefront) on FOUR wavefronts, one per SIMD, each with the full register file.
//
// Why a second tile shape: in the 128-row kernel every weight is dequantised once per 128 activation rows and every
// activation operand read from LDS feeds four MFMAs; the dequantiser's vector instructions and the LDS reads cost power,
// and on this part the matrix pipeline's clock is set by power.  Here
//   * a work-group of 4 wavefronts owns 256 activation rows x 256 weight rows; wavefront w owns weight rows 64 w ..
//     64 w + 63 (four MFMA tiles) against all 256 activation rows (sixteen MFMA tiles): 256 accumulator registers, kept
//     in the accumulation half of the register file, and per MFMA half the dequantiser arithmetic and half the LDS
//     operand traffic of the 128-row kernel;
//   * a step is 128 values of K in two ring slots of 80 KB (activation tile [256 rows][256 B] + the four wavefronts'
//     packed weights): all of the CU's LDS.  Scales and zero points therefore do not pass through LDS: every lane
//     gathers the two values of its own weight rows for the next step straight into registers (eight 2-byte loads per
//     wavefront and step, issued ahead of the step's activation loads, waited for half a step later);
//   * one barrier per step; the waits count loads exactly (vmcnt(4) at the top of a step leaves the packed weights
//     of the step after next in flight, vmcnt(16) in the middle leaves the next activation tile), every step issues the
//     same number of loads (past the end: the last step again, into a slot nobody reads).
// The k assignment inside a step, both LDS tile layouts and their swizzles are the streaming kernel's (gemm_addr.h:
// sw_*, sa_* with sixteen activation tiles).  Zero-point tensors: the kernel holds both step loops (the accumulators sit in
// the accumulation registers either way, so two loops do not cost spills) and runs folded while the zero points of the
// step ahead are small integers; from the first step whose zero points are not, the rest runs unfolded (on integral
// zero points the two dequantisers give the same bits, so the switch does not show in the result).
#include "panel256.h"

namespace tlq {

void launch_splitk_reduce(const float* partial, void* C, int64_t M, int64_t N, int split, int out_dtype, hipStream_t st);

namespace {

template <typename T, int LAYOUT, int ZM>
__global__ __launch_bounds__(256, 1) void w4a16_panel256_kernel(const T* __restrict__ A, const uint8_t* __restrict__ Wp,
                                                               const T* __restrict__ scales, const T* __restrict__ zeros,
                                                               void* __restrict__ C, float* __restrict__ partial, int M, int N, int K,
                                                               int gshift, float zero_scalar, int out_dtype, int slice_steps,
                                                               int blocks, int band_rows) {
  typedef Panel2Cfg Cfg;
  typedef Panel2Mma<T> Mma;
  constexpr int TM = Cfg::TM, TN = Cfg::TN, LA = Cfg::LA;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileCoord tc = tile_of_block<Cfg::BM, Cfg::BN>(blocks, M, N, band_rows);  // batch = K slice
  const int m0 = tc.m0, n0 = tc.n0, slice = tc.batch;
  const int steps_total = K >> 7;
  const int step0 = slice * slice_steps;
  const int steps = steps_total - step0 < slice_steps ? steps_total - step0 : slice_steps;
  const int groups = K >> gshift;

  // ---- sources of the loads: the row block of every load instruction sits in the lane offset (16 weight rows or 4
  // activation rows per instruction; N % 16 == 0, blocks past a matrix repeat its last, activation rows past it its last row; a matrix spans less
  // than 4 GiB), so that a step's loads share one scalar base and issuing one costs two instructions -- with one
  // wavefront per SIMD nothing else hides address arithmetic.
  uint32_t voff_a[LA], voff_w[TN], voff_sc[TN];
#pragma unroll
  for (int j = 0; j < LA; ++j)
    voff_a[j] = addr::panel2_a_voff(lane, wave, j, m0, M, K);
#pragma unroll
  for (int tn = 0; tn < TN; ++tn) {
    voff_w[tn] = (uint32_t)addr::panel_w_block(wave, tn, n0, N, K) + addr::panel_w_lane(lane, K);
    voff_sc[tn] = (uint32_t)addr::panel2_sc_block(wave, tn, n0, N, groups) + addr::panel2_sc_lane(lane, groups, gshift);
  }
  typename Mma::acc_t acc[TN][TM];
  panel256_steps<T, LAYOUT, ZM>(smem, A, Wp, scales, zeros, voff_a, voff_w, voff_sc, step0, steps, gshift, zero_scalar, acc);

  // lane (r16, q) holds C[m = m0 + 16 tm + r16][n = n0 + 64 wave + 16 tn + 4 q + 0..3]
  const bool split = slice_steps < steps_total;
  EpiFloat::Params pe{split ? (void*)partial : C, N, (int64_t)M * N, split ? TLQ_F32 : out_dtype};
  const EpiFloat epi(pe, split ? slice : 0);
  static_assert(Cfg::WAVES * TM * 16 * kStageBytes <= Cfg::LDS, "the staging areas of the wavefronts fit the ring");
  // (everyone is past the last step: the ring becomes the output staging area)
  write_tile<EpiFloat, TM, TN>(epi, acc, smem + wave * (TM * 16 * kStageBytes), lane, m0, n0 + wave * (16 * TN), M, N);
}

}  // namespace

thread_local int g_panel2_slice_steps = 0;  // tuning and tests: steps of 128 values of K per slice (0: the plan's own)

// Launch geometry.  ok = the kernel applies.
struct Panel2Plan {
  bool ok;
  int tiles_m, tiles_n, split, slice_steps;
};
Panel2Plan w4a16_panel256_plan(int64_t M, int64_t N, int64_t K, int64_t group, int cus) {
  Panel2Plan p{false, 0, 0, 0, 0};
  if (M < 1 || N < 1 || K < 128 || K % 128 != 0 || group < 32 || (group & (group - 1)) != 0 || K % group != 0) return p;
  if (N % 16 != 0 || M % 4 != 0) return p;  // a direct load (16 weight rows, 4 activation rows) lies inside a matrix or outside
  if (M >= ((int64_t)1 << 30) || N >= ((int64_t)1 << 30)) return p;
  p.tiles_m = (int)ceil_div(M, (int64_t)Panel2Cfg::BM);
  p.tiles_n = (int)ceil_div(N, (int64_t)Panel2Cfg::BN);
  const int steps_total = (int)(K / 128);
  // a slice is a whole number of groups or, with groups longer than a slice (one scale per weight row, say), a power-of-two
  // part of one group: the kernel takes every step's group from the step's position in K
  const int unit = group > 128 ? (int)(group / 128) : 1;
  auto whole_or_part = [&](int64_t steps) {
    if (steps >= unit) return ceil_div(steps, (int64_t)unit) * unit;
    int64_t part = 1;
    while (part < steps) part *= 2;
    return part;
  };
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (cus <= 0) cus = 256;
  int64_t ss = steps_total;
  if (g_panel2_slice_steps > 0) {
    ss = whole_or_part((int64_t)g_panel2_slice_steps);
  } else if (tiles * 2 <= cus) {
    // K slices only where the tiles leave most of the machine idle: the cut that fills it best with slices of 16 steps or more
    double best = (double)ceil_div(tiles, (int64_t)cus) * (steps_total + 8);
    for (int64_t want = 2; want <= 16; ++want) {
      int64_t cand = whole_or_part(ceil_div((int64_t)steps_total, want));
      if (cand < 16 || cand >= steps_total) continue;
      const int64_t sl = ceil_div((int64_t)steps_total, cand);
      const double t = (double)ceil_div(tiles * sl, (int64_t)cus) * (double)(cand + 8) + (double)sl * (double)M * (double)N * 4.0 / 3e6 / 3.0;
      if (t < best * 0.95) best = t, ss = cand;
    }
  }
  if (ss > steps_total) ss = steps_total;
  if (ss < 1) return p;
  p.slice_steps = (int)ss;
  p.split = (int)ceil_div((int64_t)steps_total, ss);
  if ((int64_t)p.split * tiles > 0x7fffffff) return p;
  p.ok = true;
  return p;
}

template <typename T, int LAYOUT, int ZM>
static int launch_panel256(const void* A, const void* Wp, const void* scales, const void* zeros, void* C, float* partial, int64_t M,
                           int64_t N, int64_t K, int gshift, float zero_scalar, int out_dtype, const Panel2Plan& p, int band_rows,
                           hipStream_t st) {
  auto kern = w4a16_panel256_kernel<T, LAYOUT, ZM>;
  constexpr int lds_bytes = Panel2Cfg::LDS;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
    if (e != hipSuccess) {
      set_error("tlq_gemm_w4a16(panel256): cannot reserve %d bytes of LDS: %s", lds_bytes, hipGetErrorString(e));
      return 1;
    }
    attr_set = true;
  }
  const unsigned blocks = (unsigned)((int64_t)p.tiles_m * p.tiles_n * p.split);
  kern<<<blocks, 256, lds_bytes, st>>>((const T*)A, (const uint8_t*)Wp, (const T*)scales, (const T*)zeros, C, partial, (int)M, (int)N,
                                       (int)K, gshift, zero_scalar, out_dtype, p.slice_steps, (int)blocks, band_rows);
  return check_launch("tlq_gemm_w4a16(panel256)", ZM == 0 ? "w4a16_panel256_kernel, zero-point tensor" : "w4a16_panel256_kernel")
             ? 0
             : 1;
}

// partial: fp32 [split][M][N] workspace, needed when the plan has more than one K slice
int gemm_w4a16_panel256(const void* A, const void* Wp, const void* scales, const void* zeros, void* C, int64_t M, int64_t N, int64_t K,
                        int64_t group, float zero_scalar, int in_dtype, int out_dtype, int w_layout, const Panel2Plan& p, float* partial,
                        hipStream_t st) {
  int gshift = 0;
  while (((int64_t)1 << gshift) < group) ++gshift;
  const int band = g_gemm_band_rows > 0 ? g_gemm_band_rows : 4;
  const bool fold_scalar = zero_folds(zero_scalar);
  int rc;
#define TLQ_PANEL3(T, LAY, ZM) launch_panel256<T, LAY, ZM>(A, Wp, scales, zeros, C, partial, M, N, K, gshift, zero_scalar, out_dtype, p, band, st)
#define TLQ_PANEL2(T, ZM) (w_layout == TLQ_W_INTERLEAVED_F16 ? TLQ_PANEL3(T, 1, ZM) : TLQ_PANEL3(T, 0, ZM))
#define TLQ_PANEL(ZM) (in_dtype == TLQ_F16 ? TLQ_PANEL2(half_t, ZM) : TLQ_PANEL2(bf16_t, ZM))
  if (zeros != nullptr)
    rc = TLQ_PANEL(0);
  else
    rc = fold_scalar ? TLQ_PANEL(1) : TLQ_PANEL(2);
#undef TLQ_PANEL
#undef TLQ_PANEL2
#undef TLQ_PANEL3
  if (rc) return rc;
  if (p.split > 1) {
    launch_splitk_reduce(partial, C, M, N, p.split, out_dtype, st);
    return check_launch("tlq_gemm_w4a16(panel256, reduce)", "splitk_reduce_kernel") ? 0 : 1;
  }
  return 0;
}

}  // namespace tlq
