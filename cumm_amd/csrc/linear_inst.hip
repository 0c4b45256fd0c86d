// Instantiations of the products of linear.h for one element type (selected with -DCUMM_ELEM=...); the type-free half
// (which kernel, and the copy of operands that do not lie on 16-byte borders) with -DCUMM_LINEAR_HOST.
#include <algorithm>

#include "launch.h"
#include "layers.h"

namespace cummhip {

#define CUMM_CAT_(a, b) a##b
#define CUMM_CAT(a, b) CUMM_CAT_(a, b)

// Up to 16 rows: two waves a workgroup from more columns on than one workgroup per CU takes, else eight.  us with two and with eight, one row,
// bf16, weights that no cache holds, k 256, 1024, 4096, 8192: 2048 columns 3.2 4.0 7.6 15.3 and 3.5 3.9 7.0 11.6, 4096 3.4 4.1 10.7 18.9 and 3.6 4.7 9.2 17.7,
// 6144 3.8 5.0 12.3 24.3 and 5.3 7.3 14.2 25.9, 8192 3.9 5.3 15.3 32.5 and 5.6 7.7 16.6 31.7, 28672 7.9 14.2 45.4 94.9 and 16.5 22.9 46.4 92.9; 16 rows and
// 8-bit operands within 5 % of the same.
constexpr int kFewWide = 4096;

#ifdef CUMM_LINEAR_HOST

// Which kernel and how many slices: the least estimated time, in us on 256 CUs.  The figures are fitted (non-negative least
// squares of the relative error, 12 % on average) to 42 k timings of 2400 random products of all three layouts, bf16: m to
// 120000, n to 16384, k to 100000.  With them the choice is 4.6 % slower than the fastest of every kernel and number of
// slices tried, on 1870 other products (fitted to those 4.2 %, but then 392 x 568 over 42200 rows takes 99 us
// instead of 46).  R: workgroups per CU, rounded up while there are one or two (one per CU: always), as they are beyond; steps of 64 k.
//   launch + R (turn + step * steps) + MB of operands and result + MB of partial sums + joining them, by R = 1, 2, more
// f16 and 8-bit operands take the same figures (k of those in pairs): 4.0 and 5.2 % slower than the fastest on 300 other forward products each.
// 64 x 64 in four waves and two stages (rows by the hundred thousand and a step or two: 119985 x 64 x 64 9.5 us against 12.7),
// or in 2 x 2 x 2 waves and three; 64 x 128 in 2 x 4, three stages; both with steps of 128 k where a CU has one workgroup; the others
// through registers.  Few rows (17 to 64; up to 16 always): 16 columns per workgroup.  What decides: up to 32 rows nearly always the kernel for few
// (31 x 2376 x 72 4.8 us against 14.1 in eight slices), above them while one round of workgroups does (60 x 5256 x 15680
// 57 us against 31); slices where tiles leave CUs idle (weight gradient 264 x 344 over 72024 rows 40 us in 16 of 64 x 128);
// 128 x 256 where the large tile leaves half of the CUs idle (4096 x 8192 x 2048 123 us, 128 x 128 142, 256 x 256 186); the large tile from about one per CU on (4096^3 103 us against 125).
struct TileFigures {
  double launch, turn, step, operands, partial, join;
};
constexpr TileFigures kTiles[6][3] = {
    {{3.003, 0, 0.2961, 0.1575, 0.6559, 2.241}, {0, 1.805, 0.2707, 0.01193, 0.6338, 1.618}, {3.626, 0.3804, 0.2655, 0.01601, 0.3635, 2.196}},      // 64 x 64, four waves
    {{0, 3.407, 0.2307, 0.0382, 0.8178, 2.341}, {0, 2.301, 0.2458, 0.00269, 0.6358, 1.569}, {4.167, 0.7239, 0.2754, 0, 0.2664, 2.387}},      // 64 x 64
    {{3.561, 0, 0.3179, 0.04139, 0.724, 2.238}, {0, 2.456, 0.3213, 0.04474, 0.5992, 0.7795}, {4.777, 1.028, 0.3715, 0.02534, 0.2561, 2.198}},      // 64 x 128
    {{4.548, 0, 0.4215, 0.03335, 0.6902, 1.861}, {0, 3.524, 0.419, 0.02631, 0.4779, 0}, {5.877, 1.281, 0.5569, 0.03775, 0.3011, 0}},      // 128 x 128
    {{0, 6.656, 0.6827, 0.03557, 0.576, 0.845}, {3.231, 4.953, 0.794, 0.02276, 0.2717, 0}, {3.231, 4.953, 0.794, 0.02276, 0.2717, 0}},      // 128 x 256
    {{0, 8.813, 1.027, 0.04948, 0.4428, 0}, {0, 5.446, 1.354, 0.03894, 0.3245, 0}, {0, 5.446, 1.354, 0.03894, 0.3245, 0}},      // 256 x 256
};
// Kernels whose launch would have too many threads are passed over; where all would, the plan is one that does not fit.
LinearPlan linear_plan(LinearLayout layout, int64_t m, int n_, int64_t k) {
  const int64_t n = n_;      // (the sums below may pass 2^31)
  const LinearPlan few = {kTileFew, 1, 0};
  const bool few_fit = linear_plan_fits(few, m, n_);
  if (layout == kResult && m <= 16 && few_fit) {      // (the estimate: the wave's steps, or the weight at 4.8 TB/s)
    return {kTileFew, 1, std::max(3.5 + 0.18 * (double)((k + 255) / 256), 2.0 + (double)n * k * 2e-6 / 4.8)};
  }
  LinearPlan best = {kTile64, 1, 0};
  double least = 1e300;
  const double operands = ((double)m * k + (double)n * k) * 2e-6, sums = (double)m * n * 4e-6;
  if (layout == kResult && m <= 64 && few_fit) {
    const bool two = m <= 32;      // blocks of 16 rows: two workgroups fit a CU, else one
    const double rounds = (double)(((n + 15) / 16 + (two ? 511 : 255)) / (two ? 512 : 256)), steps = (double)((k + 255) / 256);
    least = two ? 1.031 + rounds * (1.989 + 0.1778 * steps) : 1.397 + rounds * (2.037 + 0.2782 * steps);
    best = {kTileFew, 1, least};
  }
  constexpr int kShape[6][3] = {{64, 64, kTile64Small}, {64, 64, kTile64}, {64, 128, kTile64x128}, {128, 128, kTile128}, {128, 256, kTile128x256}, {256, 256, kTile256}};
  bool fits[6];
  for (int t = 0; t < 6; ++t) fits[t] = linear_plan_fits({kShape[t][2], 1, 0}, m, n_);
  const int64_t tiles = ((m + 63) / 64) * ((n + 63) / 64);      // (more than fill the device many times over need no slices)
  for (int slices = 1; slices <= 256; slices *= 2) {
    if (slices > 1 && (k / slices < 128 || tiles * slices > 16384)) break;
    const double steps = (double)(((k + slices - 1) / slices + 63) / 64);
    for (int t = 0; t < 6; ++t) {
      if (!fits[t]) continue;
      const double wgs = (double)((m + kShape[t][0] - 1) / kShape[t][0]) * (double)((n + kShape[t][1] - 1) / kShape[t][1]) * slices;
      const int regime = wgs <= 256 ? 0 : (wgs <= 512 ? 1 : 2);
      const double rounds = regime < 2 ? regime + 1.0 : (t >= 4 ? (double)(int64_t)((wgs + 255) / 256) : wgs / 256);
      const TileFigures &f = kTiles[t][regime];
      const double us = f.launch + rounds * (f.turn + f.step * steps) + f.operands * (operands + (slices == 1 ? sums / 2 : 0.0)) +
                        (slices == 1 ? 0.0 : f.partial * sums * slices + f.join);
      if (us < least) least = us, best = {kShape[t][2], slices, us};
    }
  }
  return best;
}

bool linear_plan_fits(const LinearPlan &plan, int64_t m, int n) {
  const auto threads = [&](int64_t tm, int64_t tn, int64_t per) { return (m + tm - 1) / tm * ((n + tn - 1) / tn) * per < (int64_t)1 << 32; };
  switch (plan.tile) {
  case kTileFew: return threads(m, 16, m > 16 ? 256 : (n > kFewWide ? 128 : 512));
  case kTile64Small: return threads(64, 64, 256);
  case kTile64: return threads(64, 64, 512);
  case kTile64x128: return threads(64, 128, 512);
  case kTile128: return threads(128, 128, 512);
  case kTile128x256: return threads(128, 256, 512);
  case kTileAny: return threads(64, 64, 256);
  default: return threads(256, 256, 512);
  }
}

// The same for operands that are not whole pieces on 16-byte borders, `copied` bytes of them: the copy and the plan for its result, or
// tiles that read them as they lie.  The copy costs a launch and what it moves; loads at odd addresses a step of 0.45 us where a
// CU has one workgroup, 0.33 where it has more (aligned ones do not bound these tiles: 2001 x 1168 -> 777 12 – 13.6 us either way).  f16, with
// the copy and as they lie: 1000 x 1001 -> 1000 14.1 us and 11.8, 15465 x 1603 -> 64 28.9 and 16.5, 5 x 2299 -> 6848 21.0 and 14.8 (two
// slices), 64 x 999 -> 16000 20.9 and 12.4, 6 x 537 -> 64 10.6 and 7.3; 4000 x 3001 -> 2000 65 and 130, 1550 x 452 -> 8048 31 and 43.
LinearPlan linear_plan_any(const LinearPlan &plan, int64_t m, int n, int64_t k, int64_t copied) {
  LinearPlan best = plan;
  best.us = plan.us + 4.0 + (double)copied * 2e-6 / 6.5;
  const double sums = (double)m * n * 4e-6;
  for (int slices = 1; slices <= 16 && (slices == 1 || k / slices >= 128); slices *= 2) {
    const double steps = (double)(((k + slices - 1) / slices + 63) / 64);
    const int64_t wgs = (m + 63) / 64 * (((int64_t)n + 63) / 64) * slices;
    const double us = 3.3 + std::max(0.45 * steps, (double)((wgs + 255) / 256) * (0.33 * steps + 0.9)) + (slices == 1 ? 0.0 : 3.9 + 0.4 * sums * slices);
    const LinearPlan any = {kTileAny, slices, us};
    if (us < best.us && linear_plan_fits(any, m, n)) best = any;
  }
  return best;
}

hipError_t launch_linear_repack(LinearRepack p, int elem_bytes, hipStream_t s) {
  int64_t wgs = 0;
  for (LinearRepack::One &o : p.of) {
    o.pieces = (o.cols * elem_bytes + 15) / 16;
    o.wgs = std::min<int64_t>((o.rows * o.pieces + 255) / 256, 1 << 20);
    wgs += o.wgs;
  }
  if (wgs == 0) return hipSuccess;
  if (elem_bytes == 1) hipLaunchKernelGGL(linear_repack_kernel<1>, dim3((unsigned)wgs), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(linear_repack_kernel<2>, dim3((unsigned)wgs), dim3(256), 0, s, p);
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
template <class T, class OUT, int RBW, int NBW, int NS, bool XT, bool YT>
static hipError_t pipe(const LinearParams &p, hipStream_t s) {
  constexpr int TM = 2 * RBW * 16, TN = 4 * NBW * 16;
  if (!counted_waits_hold<linear_pipe_kernel<T, OUT, 2, 4, RBW, NBW, NS, XT, YT>>()) return hipErrorNotSupported;
  const int tiles_m = (int)((p.m + TM - 1) / TM), tiles_n = (p.n + TN - 1) / TN;
  hipLaunchKernelGGL((linear_pipe_kernel<T, OUT, 2, 4, RBW, NBW, NS, XT, YT>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)p.slices), dim3(512), 0, s, p,
                     tiles_m, tiles_n);
  return hipGetLastError();
}
template <class T, class OUT, bool XT, bool YT>
static hipError_t large(const LinearParams &p, hipStream_t s) {
  if (!counted_waits_hold<linear_large_kernel<T, OUT, XT, YT>>()) return hipErrorNotSupported;
  const int tiles_m = (int)((p.m + 255) / 256), tiles_n = (p.n + 255) / 256;
  hipLaunchKernelGGL((linear_large_kernel<T, OUT, XT, YT>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)p.slices), dim3(512), 0, s, p, tiles_m, tiles_n);
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
  const auto wgs = [&](int64_t tm, int tn) { return (p.m + tm - 1) / tm * ((p.n + tn - 1) / tn) * p.slices; };
  switch (plan.tile) {
  case kTileFew:
    if constexpr (!XT && !YT) {
      if (p.m <= 16) return p.n > kFewWide ? few<T, OUT, 2, 1, 2, 4>(p, s) : few<T, OUT, 8, 1, 2, 3>(p, s);
      if (p.m <= 32) return few<T, OUT, 4, 2, 2, 3>(p, s);
      if (p.m <= 64) return few<T, OUT, 4, 4, 2, 3>(p, s);
    }
    return e;
  case kTile64Small: e = ring<T, OUT, 2, 2, 1, 2, 2, 2, 2, XT, YT>(p, s); break;
  // (one workgroup per CU: steps of 128 k, twice as much on its way: 1024 x 4096 x 1024 20.4 -> 16.0 us, 332 x 3648 x 1579 18.5 -> 15.7)
  case kTile64:
    if (wgs(64, 64) <= 256) e = ring<T, OUT, 2, 2, 2, 2, 2, 4, 4, XT, YT>(p, s);
    else e = ring<T, OUT, 2, 2, 2, 2, 2, 2, 3, XT, YT>(p, s);
    break;
  case kTile64x128:
    if (wgs(64, 128) <= 256) e = ring<T, OUT, 2, 4, 1, 2, 2, 4, 3, XT, YT>(p, s);
    else e = ring<T, OUT, 2, 4, 1, 2, 2, 2, 3, XT, YT>(p, s);
    break;
  case kTile128:      // (three stages where a CU has one workgroup: 2048^3 21.9 us against 24.9; two of two: 8192 x 1024 x 2048 39 against 48)
    if (wgs(128, 128) <= 256) e = pipe<T, OUT, 4, 2, 3, XT, YT>(p, s);
    else e = pipe<T, OUT, 4, 2, 2, XT, YT>(p, s);
    break;
  case kTile128x256: e = pipe<T, OUT, 4, 4, 3, XT, YT>(p, s); break;
  case kTileAny:
    if constexpr (!XT && !YT) {
      const int tiles_m = (int)((p.m + 63) / 64), tiles_n = (p.n + 63) / 64;
      hipLaunchKernelGGL((linear_any_kernel<T, OUT, 2, 2, 2, 2, 2, 2>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)p.slices), dim3(256), 0, s, p, tiles_m, tiles_n);
      e = hipGetLastError();
    }
    break;
  case kTile256: e = large<T, OUT, XT, YT>(p, s); break;
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
