// Instantiations of the products of linear.h for one element type (selected with -DCUMM_ELEM=...); the type-free half
// (which kernel, and the copy of operands that do not lie on 16-byte borders) with -DCUMM_LINEAR_HOST.
#include <algorithm>

#include "launch.h"
#include "layers.h"

namespace cummhip {

#define CUMM_CAT_(a, b) a##b
#define CUMM_CAT(a, b) CUMM_CAT_(a, b)

#ifdef CUMM_LINEAR_HOST

LinearPlan linear_plan(LinearLayout layout, int64_t m, int n, int64_t k) {
  if (layout == kResult && m <= 64) return {kTileFew, 1};
  const auto tiles = [&](int tm, int tn) { return ((m + tm - 1) / tm) * (int64_t)((n + tn - 1) / tn); };
  const double kd = (double)k;
  LinearPlan best = {kTile64, 1};
  double least = 1e300;
  for (int slices = 1; slices <= 256; slices *= 2) {
    if (slices > 1 && k / slices < 256) break;
    const double ks = kd / slices;
    const double join = slices == 1 ? 0.0 : 4.0 + (double)m * n * 4.0 * (2.0 * slices) / 4e6;
    const auto per_cu = [&](int tm, int tn) { return (double)((tiles(tm, tn) * slices + 255) / 256); };
    const auto consider = [&](int tile, double us) {
      if (us + join < least) least = us + join, best = {tile, slices};
    };
    const double n64 = per_cu(64, 64), n128 = per_cu(128, 128), n256 = per_cu(256, 256);
    consider(kTile64, n64 == 1 ? 3.7 + 0.0040 * ks : (n64 == 2 ? 4.9 + 0.0063 * ks : 2.4 + n64 * (1.12 + 0.0031 * ks)));
    if (n128 == 1) consider(kTile128Deep, std::max(9.4, 7.0 + 0.0072 * ks));
    else consider(kTile128, n128 == 2 ? 8.2 + 0.0122 * ks : n128 * (3.9 + 0.0077 * ks));
    consider(kTile256, std::max(2.0 + n256 * (14.8 + 0.0235 * ks), 8.5 + 0.0255 * n256 * ks));
  }
  return best;
}

hipError_t launch_linear_repack(void *to, const void *from, int64_t rows, int64_t cols, int64_t ld, int64_t to_ld, int elem_bytes, hipStream_t s) {
  const int64_t pieces = (cols * elem_bytes + 15) / 16;
  const int64_t wgs = std::min<int64_t>((rows * pieces + 255) / 256, 1 << 20);
  if (wgs == 0) return hipSuccess;
  if (elem_bytes == 1) hipLaunchKernelGGL(linear_repack_kernel<1>, dim3((unsigned)wgs), dim3(256), 0, s, (v4i *)to, from, rows, cols, ld, pieces, to_ld);
  else hipLaunchKernelGGL(linear_repack_kernel<2>, dim3((unsigned)wgs), dim3(256), 0, s, (v4i *)to, from, rows, cols, ld, pieces, to_ld);
  return hipGetLastError();
}

#else

template <class T, class OUT>
static hipError_t join(const LinearParams &p, hipStream_t s) {
  if (p.slices == 1) return hipSuccess;
  const int64_t items = p.m * ((p.n + 7) / 8);
  constexpr bool S8OP = Elem<T>::kBytes == 1;
  if (p.slices >= 16) hipLaunchKernelGGL((linear_join_kernel<OUT, S8OP, 8>), dim3((unsigned)((items + 31) / 32)), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((linear_join_kernel<OUT, S8OP, 1>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, p);
  return hipGetLastError();
}

// (the kernels count their loads: see counted_waits_hold)
template <class T, class OUT, int WM, int WN, int WK, int RBW, int NBW, int KS, int NS, bool XT, bool YT>
static hipError_t ring(const LinearParams &p, hipStream_t s) {
  constexpr int TM = WM * RBW * 16, TN = WN * NBW * 16;
  if (!counted_waits_hold<linear_ring_kernel<T, OUT, WM, WN, WK, RBW, NBW, KS, NS, XT, YT>>()) return hipErrorNotSupported;
  const int tiles_m = (int)((p.m + TM - 1) / TM), tiles_n = (p.n + TN - 1) / TN;
  hipLaunchKernelGGL((linear_ring_kernel<T, OUT, WM, WN, WK, RBW, NBW, KS, NS, XT, YT>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)p.slices),
                     dim3(WM * WN * WK * 64), 0, s, p, tiles_m, tiles_n);
  return hipGetLastError();
}
template <class T, class OUT, bool XT, bool YT>
static hipError_t pipe(const LinearParams &p, hipStream_t s) {
  if (!counted_waits_hold<linear_pipe_kernel<T, OUT, 2, 4, 8, 4, 4, XT, YT>>()) return hipErrorNotSupported;
  const int tiles_m = (int)((p.m + 255) / 256), tiles_n = (p.n + 255) / 256;
  hipLaunchKernelGGL((linear_pipe_kernel<T, OUT, 2, 4, 8, 4, 4, XT, YT>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)p.slices), dim3(512), 0, s, p,
                     tiles_m, tiles_n);
  return hipGetLastError();
}
template <class T, class OUT, int W, int MB, int KS, int NS>
static hipError_t few(const LinearParams &p, hipStream_t s) {
  if (!counted_waits_hold<linear_few_kernel<T, OUT, W, MB, KS, NS>>()) return hipErrorNotSupported;
  hipLaunchKernelGGL((linear_few_kernel<T, OUT, W, MB, KS, NS>), dim3((unsigned)((p.n + 15) / 16)), dim3(W * 64), 0, s, p);
  return hipGetLastError();
}

template <class T, class OUT, bool XT, bool YT>
static hipError_t launch_layout(const LinearPlan &plan, const LinearParams &p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  switch (plan.tile) {
  case kTileFew:
    if constexpr (!XT && !YT) {
      if (p.m <= 16) return few<T, OUT, 4, 1, 2, 3>(p, s);
      if (p.m <= 32) return few<T, OUT, 4, 2, 2, 3>(p, s);
      if (p.m <= 64) return few<T, OUT, 4, 4, 2, 3>(p, s);
    }
    return e;
  case kTile64: e = ring<T, OUT, 2, 2, 2, 2, 2, 2, 3, XT, YT>(p, s); break;
  case kTile128: e = ring<T, OUT, 2, 4, 1, 4, 2, 2, 2, XT, YT>(p, s); break;
  case kTile128Deep: e = ring<T, OUT, 2, 4, 1, 4, 2, 2, 4, XT, YT>(p, s); break;
  case kTile256: e = pipe<T, OUT, XT, YT>(p, s); break;
  }
  return e == hipSuccess ? join<T, OUT>(p, s) : e;
}

#define CUMM_LAUNCH_NAME CUMM_CAT(launch_linear_, CUMM_NAME)
#ifdef CUMM_LINEAR_S8
hipError_t launch_linear_s8(bool bf16, const LinearPlan &plan, const LinearParams &p, hipStream_t s) {
  return bf16 ? launch_layout<S8, BF16, false, false>(plan, p, s) : launch_layout<S8, F16, false, false>(plan, p, s);
}
#else
hipError_t CUMM_LAUNCH_NAME(LinearLayout layout, const LinearPlan &plan, const LinearParams &p, hipStream_t s) {
  using T = CUMM_ELEM;
  if (layout == kGradInput) return launch_layout<T, T, true, false>(plan, p, s);
  if (layout == kGradWeight) return launch_layout<T, T, true, true>(plan, p, s);
  return launch_layout<T, T, false, false>(plan, p, s);
}
#endif
#endif

}  // namespace cummhip
