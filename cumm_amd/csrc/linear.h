// Matrix product of rows with a weight, bias, activation and residual in its epilogue,
//   out[m][n] = act( sum_k x[m][k] w[n][k] + bias[n] ) + residual[m][n],
// and the two products of its backward pass, on matrix cores:
//   D[m][n] = sum_k Y[m][k] X[n][k]      X, Y contiguous along k, or along their rows (XT, YT)
//     result            Y = x,             X = w
//     grad_x            Y = dz [m][n],     X = w  read along its rows (the contraction is over n)
//     grad_weight       Y = dz, X = x, both along their rows (the contraction is over m)
// Operands lie in LDS as densegemm_lds.h has them (DenseOperand: permuted 16-byte chunks, direct-to-LDS
// loads, hand-counted waits).  What is different here:
//   * addresses are 64 bits: a tile's descriptor begins at its own first row and moves by a step's bytes, so
//     that no operand has a size limit; offsets inside a tile's step stay below 2^31 bytes (checked on the host);
//   * 8-bit operands are pairs of bytes to the copies and the LDS layout, only the products know them;
//   * operands that are not whole 16-byte pieces on 16-byte borders are copied, or read as they lie (linear_any_kernel);
//   * the contraction can be cut into slices (grid.y), whose 32-bit sums a second kernel adds up in order;
//   * the epilogue below.
#pragma once
#include "densegemm_lds.h"
#include "rows.h"

namespace cummhip {

enum LinearAct { kActNone = 0, kActRelu = 1, kActSigmoid = 2, kActLeakyRelu = 3, kActSilu = 4, kActGelu = 5, kActGeluTanh = 6 };

struct LinearParams {
  const void *X, *Y;       // operand indexed by n, by m
  int64_t ldx, ldy;        // bytes between rows (XT, YT: between k slices)
  int64_t m;
  int32_t n;
  int64_t k;               // of two bytes each: elements, pairs of 8-bit ones
  void *out;
  int64_t ldo;             // elements, as ldr and ldp
  const void *bias;        // [n] in the output's type, f32 with 8-bit operands; NULL = none
  const void *residual;    // [m, n] or NULL
  int64_t ldr;
  void *pre;               // [m, n]: what the activation gets, for the backward pass; NULL = not wanted
  int64_t ldp;
  const float *y_scale, *x_scale;   // 8-bit operands: [m], [n]
  int32_t act;
  float slope;
  void *partial;           // slices > 1: [slices][m][n8] 32-bit sums, n8 = n rounded up to 8
  int32_t slices;
  int32_t row_bytes;       // linear_any_kernel: k in bytes
};

// ---- the epilogue: values v[8] are consecutive columns n .. n + 7 of a row

// log2(e), and of 2 sqrt(2 / pi) (z + 0.044715 z^3): the tanh form of the gelu is z times the logistic function of that
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kGeluA = 2.30220819813f, kGeluB = 0.10294324038f;      // kLog2e * 2 sqrt(2/pi), the same * 0.044715

__device__ __forceinline__ float logistic_of_exponent(float t) {      // 1 / (1 + 2^t)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}
// The smaller tail of the normal distribution beyond |z|, and e^(-z^2 / 2) beside it.  Their quotient falls slowly, from 1.25 to 1 / |z|; a
// polynomial in t = 1 / (1 + 0.289 |z|) follows it to 1.6e-4 of itself up to |z| = 14, where the tail ends in the denormals, and so that the
// tail is off by less than 4.7e-8 everywhere (linear programming for the least of both errors at once; in 32 bits 2e-7 and 1.6e-4).  A
// negative argument's gelu is z times the tail: what it needs is the former, below the half step of f16 and bf16.
__device__ __forceinline__ float normal_tail(float z, float *e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.289f, __builtin_fabsf(z), 1.0f));
  // (its coefficients over the root of 2 pi)
  float poly = __builtin_fmaf(-0.09064557f, t, 0.2949497f);
  poly = __builtin_fmaf(poly, t, -0.10590875f);
  poly = __builtin_fmaf(poly, t, 0.18663533f);
  poly = __builtin_fmaf(poly, t, 0.09830108f);
  poly = __builtin_fmaf(poly, t, 0.1166682f);
  *e = __builtin_amdgcn_exp2f(z * (z * (-0.5f * kLog2e)));
  return poly * t * *e;
}

// The activation is uniform: one dispatch for a lane's values.  NaN stays NaN.
template <int N>
__device__ __forceinline__ void linear_act(float (&v)[N], int act, float slope) {
  switch (act) {
  case kActRelu:
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    break;
  case kActLeakyRelu:
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? v[i] * slope : v[i];
    break;
  case kActSigmoid:
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = logistic_of_exponent(-kLog2e * v[i]);
    break;
  case kActSilu:
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= logistic_of_exponent(-kLog2e * v[i]);
    break;
  case kActGeluTanh:
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= logistic_of_exponent(-v[i] * __builtin_fmaf(kGeluB, v[i] * v[i], kGeluA));
    break;
  case kActGelu:
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float e;
      const float tail = normal_tail(v[i], &e);
      v[i] *= v[i] < 0.0f ? tail : 1.0f - tail;
    }
    break;
  default: break;
  }
}

// the derivative of a smooth activation where its argument is z
__device__ __forceinline__ float linear_act_slope(float z, int act) {
  switch (act) {
  case kActSigmoid: {
    const float p = logistic_of_exponent(-kLog2e * z);
    return p * (1.0f - p);
  }
  case kActSilu: {
    const float p = logistic_of_exponent(-kLog2e * z);
    // (beyond |z| = 128 p is 0 or 1; an infinite z - any that the type it is kept in cannot hold - would be infinity times zero)
    const float zc = __builtin_amdgcn_fmed3f(z, -128.0f, 128.0f);
    return p * __builtin_fmaf(zc, 1.0f - p, 1.0f);
  }
  case kActGeluTanh: {
    const float p = logistic_of_exponent(-z * __builtin_fmaf(kGeluB, z * z, kGeluA));
    // z p(u(z)): p + z p (1 - p) u', u' = 2 sqrt(2/pi) (1 + 3 * 0.044715 z^2); beyond |z| = 16, where p is 0 or 1, the
    // cubic term would be infinite times zero
    const float zc = __builtin_amdgcn_fmed3f(z, -16.0f, 16.0f);
    const float du = __builtin_fmaf(0.21406572f * zc, zc, 1.59576912f);
    return __builtin_fmaf(zc * p * (1.0f - p), du, p);
  }
  case kActGelu: {
    float e;
    const float tail = normal_tail(z, &e);
    const float zc = __builtin_amdgcn_fmed3f(z, -16.0f, 16.0f);      // (an infinite one times zero, else)
    return __builtin_fmaf(zc * 0.39894228040143268f, e, z < 0.0f ? tail : 1.0f - tail);
  }
  default: return 1.0f;
  }
}

// Eight of them, multiplied into g: one branch for all.  Those with a kink choose: where nothing passes there is no product, an
// infinite gradient times zero is not NaN; the gradient of an argument that is NaN passes.
__device__ __forceinline__ void linear_act_slopes(float (&g)[8], const v4f &lo, const v4f &hi, int act, float slope) {
  const auto all = [&](auto one) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] *= linear_act_slope(e < 4 ? lo[e] : hi[e - 4], decltype(one)::value);
  };
  switch (act) {
  case kActRelu:
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = (e < 4 ? lo[e] : hi[e - 4]) <= 0.0f ? 0.0f : g[e];
    break;
  case kActLeakyRelu:
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = (e < 4 ? lo[e] : hi[e - 4]) <= 0.0f ? g[e] * slope : g[e];
    break;
  case kActSigmoid: all(std::integral_constant<int, kActSigmoid>{}); break;
  case kActSilu: all(std::integral_constant<int, kActSilu>{}); break;
  case kActGelu: all(std::integral_constant<int, kActGelu>{}); break;
  case kActGeluTanh: all(std::integral_constant<int, kActGeluTanh>{}); break;
  default: break;
  }
}

// Bias of columns n .. n + 7, and what the accumulators are multiplied by (8-bit operands)
template <class OUT, bool S8>
__device__ __forceinline__ void linear_columns(const LinearParams &p, int n, float (&bias)[8], float (&scale)[8]) {
  const int count = p.n - n;
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = 0.0f;
  if constexpr (S8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) scale[e] = e < count ? p.x_scale[n + e] : 0.0f;
    if (p.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[e] = e < count ? reinterpret_cast<const float *>(p.bias)[n + e] : 0.0f;
    }
  } else {
    if (p.bias != nullptr && count > 0) {
      Piece<OUT> b;
      b.load(p.bias, n, count);
      b.values(bias);
    }
  }
}

// One row's eight columns out of sums: the whole epilogue
template <class OUT, bool S8, bool NT>
__device__ __forceinline__ void linear_finish8(const LinearParams &p, int64_t m, int n, float (&v)[8], const float (&bias)[8], const float (&scale)[8]) {
  const int count = p.n - n;
  Piece<OUT> piece, add;
  add.raw = v4i{0, 0, 0, 0};
  if (p.residual != nullptr) add.load(p.residual, m * p.ldr + n, count);
  const float row = S8 ? p.y_scale[m] : 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = S8 ? __builtin_fmaf(v[e] * row, scale[e], bias[e]) : v[e] + bias[e];
  if (p.pre != nullptr) {
    piece.round(v);
    piece.template store<NT>(p.pre, m * p.ldp + n, count);
  }
  linear_act(v, p.act, p.slope);
  float r[8];
  add.values(r);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += r[e];
  piece.round(v);
  piece.template store<NT>(p.out, m * p.ldo + n, count);
}

// A wave's accumulators, RBW x NBW blocks of 16 x 16 from row m_wave, column n_wave on.  Lane (q, i) holds four columns
// of each block, of row i.  They go through the wave's share of LDS (BYTES of it, CHUNK row blocks at a time) and come
// back as eight consecutive columns a lane: whole lines of 64 or 128 bytes per row and store, and a loop over rows instead
// of an epilogue written out for every accumulator, which needs more registers than the large tile leaves.  Rows are
// [row][16 or 8 units of four columns], units permuted by the row: neither side meets a bank twice.  The residual and the
// rows' scales are fetched a group of rows ahead.
template <class OUT, bool S8, int RBW, int NBW, bool XT, bool NT, int BYTES, class AccV>
__device__ __forceinline__ void linear_epilogue(const LinearParams &p, const AccV (&acc)[RBW][NBW], int64_t m_wave, int n_wave, int lane, char *lds,
                                                int slice) {
  constexpr int UNITS = NBW * 4, PIECES = NBW * 2, ROWS = 64 / PIECES;      // ROWS at a time
  constexpr int FIT = BYTES / (NBW * 1024), CHUNK = FIT >= RBW ? RBW : (FIT >= 4 ? 4 : (FIT >= 2 ? 2 : 1));
  constexpr int TIMES = CHUNK * 16 / ROWS, GROUP = TIMES < 4 ? TIMES : 4, GROUPS = TIMES / GROUP, ALL = RBW / CHUNK * GROUPS;
  static_assert((NBW == 2 || NBW == 4) && FIT >= 1 && RBW % CHUNK == 0 && TIMES % GROUP == 0, "row blocks of a chunk");
  const int i = lane & 15, q = lane >> 4;
  const int piece = lane % PIECES, sub = lane / PIECES, n = n_wave + piece * 8, count = p.n - n;
  const bool in_n = count > 0;
  AccV *own = reinterpret_cast<AccV *>(lds);
  const auto park = [&](int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < CHUNK; ++b)
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) {
        const int unit = XT ? nb * 4 + q : (nb >> 1) * 8 + q * 2 + (nb & 1);
        own[(b * 16 + i) * UNITS + (unit ^ (i & (UNITS - 1)))] = acc[chunk * CHUNK + b][nb];
      }
    asm volatile("" ::: "memory");      // (other lanes' units: written above, in order)
  };
  const auto take = [&](int r, AccV &a, AccV &b) __attribute__((always_inline)) {
    const AccV *at = own + r * UNITS;
    a = at[(2 * piece) ^ (r & (UNITS - 1))];
    b = at[(2 * piece + 1) ^ (r & (UNITS - 1))];
  };
  if (p.partial != nullptr) {      // 32-bit sums of this slice (8-bit operands: whole numbers)
    const int64_t n8 = (p.n + 7) & ~7;
    v4i *to = reinterpret_cast<v4i *>(p.partial) + ((int64_t)slice * p.m * n8 + n) / 4;
#pragma unroll
    for (int chunk = 0; chunk < RBW / CHUNK; ++chunk) {
      park(chunk);
#pragma unroll 4
      for (int r = sub; r < CHUNK * 16; r += ROWS) {
        AccV a, b;
        take(r, a, b);
        const int64_t m = m_wave + chunk * CHUNK * 16 + r;
        if (m < p.m && in_n) {
          to[m * n8 / 4] = __builtin_bit_cast(v4i, a);
          to[m * n8 / 4 + 1] = __builtin_bit_cast(v4i, b);
        }
      }
      asm volatile("" ::: "memory");
    }
    return;
  }
  // (the residual past the L2s, whose lines the other workgroups' steps want, where there are steps: 4096 x 8192 x 2048 131.7 ->
  // 125.8 us, 8192^3 793 -> 754; 4096 x 4096 x 256 the other way, 23.1 -> 25.6)
  const bool past = NT && p.k >= 1024;
  Piece<OUT> add[GROUP];
  float row[GROUP];
  const auto fetch = [&](int group) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < GROUP; ++j) {
      const int64_t m = m_wave + (group * GROUP + j) * ROWS + sub;
      const bool in = m < p.m && in_n && group < ALL;
      add[j].raw = v4i{0, 0, 0, 0};
      row[j] = 0.0f;
      if (p.residual != nullptr && in) {
        if (past) add[j].template load<true>(p.residual, m * p.ldr + n, count);
        else add[j].load(p.residual, m * p.ldr + n, count);
      }
      if (S8 && in) row[j] = p.y_scale[m];
    }
  };
  fetch(0);
  float bias[8], scale[8];
  linear_columns<OUT, S8>(p, n, bias, scale);
#pragma unroll
  for (int chunk = 0; chunk < RBW / CHUNK; ++chunk) {
    park(chunk);
#pragma unroll 1
    for (int g = 0; g < GROUPS; ++g) {
      float v[GROUP * 8], r[GROUP * 8];
      const int64_t m0 = m_wave + (chunk * GROUPS + g) * GROUP * ROWS + sub;
#pragma unroll
      for (int j = 0; j < GROUP; ++j) {
        AccV a, b;
        take((g * GROUP + j) * ROWS + sub, a, b);
        float t[8];
        add[j].values(t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = (float)(e < 4 ? a[e & 3] : b[e & 3]);
          v[j * 8 + e] = S8 ? __builtin_fmaf(z * row[j], scale[e], bias[e]) : z + bias[e];
          r[j * 8 + e] = t[e];
        }
      }
      fetch(chunk * GROUPS + g + 1);
      const auto store = [&](void *base, int64_t ld) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
          float t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = v[j * 8 + e];
          Piece<OUT> out;
          out.round(t);
          const int64_t m = m0 + j * ROWS;
          if (m < p.m && in_n) {
            if (NT && ld % 64 == 0) out.template store<true>(base, m * ld + n, count);
            else out.store(base, m * ld + n, count);
          }
        }
      };
      if (p.pre != nullptr) store(p.pre, p.ldp);
      linear_act(v, p.act, p.slope);
#pragma unroll
      for (int e = 0; e < GROUP * 8; ++e) v[e] += r[e];
      store(p.out, p.ldo);
    }
    asm volatile("" ::: "memory");
  }
}

// ---- operands

// One operand of a tile, as DenseOperand lays it out, behind a descriptor that moves along k, BK of it a step.  What a
// chunk of 16 bytes holds behind the end of k or of the rows has to be there and, where both operands reach it, zero:
// the host sees to that (linear_repack_kernel).
template <int ROWS, int KS, int WAVES, bool TR, int SLAB_BLOCKS, bool WIDE_ORDER>
struct LinearOperand : DenseOperand<ROWS, KS, WAVES, TR, SLAB_BLOCKS, WIDE_ORDER> {
  using Base = DenseOperand<ROWS, KS, WAVES, TR, SLAB_BLOCKS, WIDE_ORDER>;
  using Base::voff;
  uint64_t at;       // where the next step begins
  int left;          // k from there on
  uint64_t step;     // bytes

  // rows first .. first + ROWS of `count`, from step `s0` on
  __device__ __forceinline__ void begin(int wave, int lane, const void *ptr, int64_t first, int64_t count, int64_t ld, int64_t k, int64_t s0) {
    const int rows_here = (int)(count - first < ROWS ? count - first : ROWS);
#pragma unroll
    for (int t = 0; t < Base::IP; ++t) {
      const int slot = (wave * Base::IP + t) * 64 + lane;
      if constexpr (TR) {
        const int e = slot / Base::CPR, c = (slot % Base::CPR) ^ Base::swap_tr(e);
        voff[t] = c * 8 < rows_here ? (uint32_t)(e * ld) + (uint32_t)c * 16u : Base::kOob;
      } else {
        const int rho = slot / Base::LPR, c = (slot % Base::LPR) ^ Base::swap_kc(rho);
        const int i = rho & 15, nb = (rho >> 4) % SLAB_BLOCKS, slab = rho / (16 * SLAB_BLOCKS);
        const int row = WIDE_ORDER ? slab * (16 * SLAB_BLOCKS) + (nb >> 1) * 32 + (i >> 2) * 8 + (nb & 1) * 4 + (i & 3) : rho;
        voff[t] = row < rows_here ? (uint32_t)(row * ld) + (uint32_t)c * 16u : Base::kOob;
      }
    }
    step = (uint64_t)(TR ? (int64_t)Base::BK * ld : (int64_t)Base::BK * 2);
    at = (uint64_t)ptr + (uint64_t)(TR ? first * 2 : first * ld) + (uint64_t)s0 * step;
    left = (int)(k - s0 * Base::BK);
  }
  // The next step, into the stage at `lds_at`; one that is not live is zeros, without traffic.  The last one takes the
  // chunks that lie behind the end of k out of the offsets, for good: a look per step, not one per load (which the
  // large tile takes 776 us for at 8192^3 instead of 759).
  v4i rsrc;
  uint32_t lds;
  __device__ __forceinline__ void aim(uint32_t lds_at, int wave, int lane, bool live) {
    rsrc = v4i{(int)(uint32_t)at, (int)((uint32_t)(at >> 32) & 0xffffu), live ? 0x7fffffff : 0, 0x00020000};
    lds = lds_at + wave * Base::IP * 1024;
    if (left < Base::BK) {
#pragma unroll
      for (int t = 0; t < Base::IP; ++t) {
        const int slot = (wave * Base::IP + t) * 64 + lane;
        const int first_k = TR ? slot / Base::CPR : ((slot % Base::LPR) ^ Base::swap_kc(slot / Base::LPR)) * 8;
        voff[t] = first_k < left ? voff[t] : Base::kOob;
      }
    }
    skip(1);
  }
  __device__ __forceinline__ void issue_one(int t) const { dma_b128(rsrc, lds + t * 1024, voff[t], 0u); }
  __device__ __forceinline__ void issue_next(uint32_t lds_at, int wave, int lane, bool live) {
    aim(lds_at, wave, lane, live);
#pragma unroll
    for (int t = 0; t < Base::IP; ++t) issue_one(t);
  }
  __device__ __forceinline__ void skip(int steps) {
    at += step * (uint64_t)steps;
    left -= steps * Base::BK;
  }
};

// The steps of a slice: whole steps, the last slice takes what is left
struct LinearSlice {
  int first, steps;
};
__device__ __forceinline__ LinearSlice linear_slice(const LinearParams &p, int step, int slice) {
  const int all = (int)((p.k + step - 1) / step), per = (all + p.slices - 1) / p.slices, first = slice * per;
  const int end = first + per < all ? first + per : all;
  return {first, end > first ? end - first : 0};
}

// Tile and slice of a workgroup: those that share an XCD take neighbouring tiles (as dense_tile has them) of the same slice, whose
// rows its L2 then fetches once (dealt out among the XCDs by tile, weight gradients over many rows read them eight times: 256 x 256
// over 100000 rows 50 us, so 31)
__device__ __forceinline__ int linear_tile(int tiles_m, int tiles_n, int *tile_m, int *tile_n) {
  const int tiles = (int)gridDim.x, all = tiles * (int)gridDim.y;
  int logical = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  if (all % 8 == 0) logical = logical % 8 * (all / 8) + logical / 8;
  const int slice = logical / tiles;
  logical -= slice * tiles;
  constexpr int GROUP = 8;
  const int per_group = GROUP * tiles_n;
  const int g = logical / per_group, r = logical % per_group;
  const int rows_here = tiles_m - g * GROUP < GROUP ? tiles_m - g * GROUP : GROUP;
  *tile_m = g * GROUP + r % rows_here;
  *tile_n = r / rows_here;
  return slice;
}

// ---- tiles of WM x WN wave tiles times WK groups of waves that share a step's slices (densegemm_lds_kernel's loop)
template <class T, class OUT, int WM, int WN, int WK, int RBW, int NBW, int KS, int NS, bool XT, bool YT>
__global__ __launch_bounds__(WM *WN *WK * 64) void linear_ring_kernel(const LinearParams p, int tiles_m, int tiles_n) {
  using E = Elem<T>;
  using AccV = typename E::AccV;
  constexpr bool S8OP = E::kBytes == 1;
  static_assert(!S8OP || (!XT && !YT), "8-bit operands are contiguous along k");
  constexpr int TM = WM * RBW * 16, TN = WN * NBW * 16;
  using OpY = LinearOperand<TM, KS, WM * WN * WK, YT, RBW, false>;
  using OpX = LinearOperand<TN, KS, WM * WN * WK, XT, NBW, !XT>;
  constexpr int STAGE = (OpY::VECS + OpX::VECS) * 16;
  constexpr int L = NS - 1;
  constexpr int WAIT_STEP = (L - 1) * (OpY::IP + OpX::IP);
  static_assert(WAIT_STEP < 64, "too many loads in flight for the counter");
  __shared__ __attribute__((aligned(16))) char ring[NS * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
  constexpr int KW = KS / WK;
  int tile_m, tile_n;
  const int of_slice = linear_tile(tiles_m, tiles_n, &tile_m, &tile_n);
  const int64_t m0 = (int64_t)tile_m * TM;
  const int n0 = tile_n * TN;
  OpY y;
  OpX x;
  const LinearSlice slice = linear_slice(p, OpY::BK, of_slice);
  y.begin(wave, lane, p.Y, m0, p.m, p.ldy, p.k, slice.first);
  x.begin(wave, lane, p.X, n0, p.n, p.ldx, p.k, slice.first);
  int y_rd[YT ? RBW : KW], x_rd[XT ? NBW : KW];
  y.offsets(lane, wm, y_rd, wk * KW);
  x.offsets(lane, wn, x_rd, wk * KW);
  AccV acc[RBW][NBW];
#pragma unroll
  for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = AccV{0, 0, 0, 0};
  const uint32_t ring_at = lds_addr(ring);
  auto issue = [&](int s, int stage) __attribute__((always_inline)) {
    const bool live = s < slice.steps;
    const uint32_t st = ring_at + (uint32_t)__builtin_amdgcn_readfirstlane(stage * STAGE);
    y.issue_next(st, wave, lane, live);
    x.issue_next(st + OpY::VECS * 16, wave, lane, live);
  };
  for (int s = 0; s < L; ++s) issue(s, s);
  int cs = 0, ls = L;
  for (int s = 0; s < slice.steps; ++s) {
    wait_vmcnt<WAIT_STEP>();
    lds_barrier();
    const char *st = ring + cs * STAGE;
    v4i yf[RBW][KW], xf[NBW][KW];
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb)
#pragma unroll
      for (int k = 0; k < KW; ++k) xf[nb][k] = OpX::fragment(st + OpY::VECS * 16 + (XT ? wk * KW * 32 * TN * 2 : 0), x_rd, k, nb);
#pragma unroll
    for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
      for (int k = 0; k < KW; ++k) yf[rb][k] = OpY::fragment(st + (YT ? wk * KW * 32 * TM * 2 : 0), y_rd, k, rb);
    issue(s + L, ls);
    cs = cs + 1 == NS ? 0 : cs + 1;
    ls = ls + 1 == NS ? 0 : ls + 1;
#pragma unroll
    for (int k = 0; k < KW; ++k)
#pragma unroll
      for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
        for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = E::mfma(xf[nb][k], yf[rb][k], acc[rb][nb]);
  }
  wait_vmcnt<0>();
  __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0): this wave has read its last stage,
  lds_barrier();                          // and so has every other
  constexpr int SHARE = NS * STAGE / (WM * WN * WK);
  if constexpr (WK == 1) {
    linear_epilogue<OUT, S8OP, RBW, NBW, XT, false, SHARE>(p, acc, m0 + wm * (RBW * 16), n0 + wn * (NBW * 16), lane, ring + wave * SHARE, of_slice);
  } else {
    // each group finishes its share of the row blocks: it adds up all groups' sums of them, in group order
    constexpr int RO = RBW / WK;
    static_assert(RBW % WK == 0 && NS * STAGE >= WM * WN * WK * RBW * NBW * 1024, "the ring holds every group's sums");
    AccV own[RO][NBW];
    AccV *park = reinterpret_cast<AccV *>(ring);   // [group][wave of the group][rb][nb][lane]
    const int wg = wave % (WM * WN);
#pragma unroll
    for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) park[(((wk * (WM * WN) + wg) * RBW + rb) * NBW + nb) * 64 + lane] = acc[rb][nb];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RO; ++r)
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) {
        AccV t = park[((wg * RBW + wk * RO + r) * NBW + nb) * 64 + lane];
#pragma unroll
        for (int g = 1; g < WK; ++g) t += park[(((g * (WM * WN) + wg) * RBW + wk * RO + r) * NBW + nb) * 64 + lane];
        own[r][nb] = t;
      }
    __syncthreads();
    linear_epilogue<OUT, S8OP, RO, NBW, XT, false, SHARE>(p, own, m0 + wm * (RBW * 16) + wk * RO * 16, n0 + wn * (NBW * 16), lane,
                                                          ring + wave * SHARE, of_slice);
  }
}

// ---- fragments double-buffered in registers: while the products of one half of a step (32 k) run on one set, those of
// the next half are read into the other.  A step is 64 k, so that a row's share of it is a whole line of 128 bytes (with
// 32 k every line is asked for twice: 8192 x 4096 x 4096 in tiles of 256 250 us instead of 210), and there are two
// stages: the loads of step s + 2 begin when the second half of step s is in registers.  Tiles of 128 x 128, two
// workgroups per CU, one of which loads, waits or stores while the other multiplies.
template <class T, class OUT, int WM, int WN, int RBW, int NBW, int NS, bool XT, bool YT>
__global__ __launch_bounds__(WM *WN * 64) void linear_pipe_kernel(const LinearParams p, int tiles_m, int tiles_n) {
  using E = Elem<T>;
  using AccV = typename E::AccV;
  constexpr bool S8OP = E::kBytes == 1;
  static_assert(!S8OP || (!XT && !YT), "8-bit operands are contiguous along k");
  constexpr int TM = WM * RBW * 16, TN = WN * NBW * 16;
  using OpY = LinearOperand<TM, 2, WM * WN, YT, RBW, false>;
  using OpX = LinearOperand<TN, 2, WM * WN, XT, NBW, !XT>;
  constexpr int STAGE = (OpY::VECS + OpX::VECS) * 16;
  constexpr int PER = OpY::IP + OpX::IP;
  __shared__ __attribute__((aligned(16))) char ring[NS * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tile_m, tile_n;
  const int of_slice = linear_tile(tiles_m, tiles_n, &tile_m, &tile_n);
  const int64_t m0 = (int64_t)tile_m * TM;
  const int n0 = tile_n * TN;
  OpY y;
  OpX x;
  const LinearSlice slice = linear_slice(p, OpY::BK, of_slice);
  y.begin(wave, lane, p.Y, m0, p.m, p.ldy, p.k, slice.first);
  x.begin(wave, lane, p.X, n0, p.n, p.ldx, p.k, slice.first);
  int y_rd[YT ? RBW : 2], x_rd[XT ? NBW : 2];
  y.offsets(lane, wm, y_rd);
  x.offsets(lane, wn, x_rd);
  AccV acc[RBW][NBW];
#pragma unroll
  for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = AccV{0, 0, 0, 0};
  const uint32_t ring_at = lds_addr(ring);
  auto issue = [&](int s, int stage) __attribute__((always_inline)) {
    const bool live = s < slice.steps;
    const uint32_t st = ring_at + (uint32_t)__builtin_amdgcn_readfirstlane(stage * STAGE);
    y.issue_next(st, wave, lane, live);
    x.issue_next(st + OpY::VECS * 16, wave, lane, live);
  };
  v4i ya[RBW], xa[NBW], yb[RBW], xb[NBW];   // the fragments of two halves
  auto read = [&](int stage, int half, v4i (&yf)[RBW], v4i (&xf)[NBW]) __attribute__((always_inline)) {
    const char *st = ring + stage * STAGE;
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) xf[nb] = OpX::fragment(st + OpY::VECS * 16, x_rd, half, nb);
#pragma unroll
    for (int rb = 0; rb < RBW; ++rb) yf[rb] = OpY::fragment(st, y_rd, half, rb);
  };
  auto products = [&](v4i (&yc)[RBW], v4i (&xc)[NBW]) __attribute__((always_inline)) {
#pragma unroll
    for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = E::mfma(xc[nb], yc[rb], acc[rb][nb]);
    // (reads and products interleaved: the scheduler would put all reads first)
    constexpr int READS = RBW * (YT ? 2 : 1) + NBW * (XT ? 2 : 1);
    constexpr int MF = RBW * NBW;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, MF / READS > 0 ? MF / READS : 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MF, 0);
  };
  for (int s = 0; s < NS; ++s) issue(s, s);
  wait_vmcnt<(NS - 1) * PER>();
  lds_barrier();
  read(0, 0, ya, xa);
  int st = 0;
  for (int s = 0; s < slice.steps; ++s) {
    const int after = st + 1 == NS ? 0 : st + 1;
    read(st, 1, yb, xb);
    products(ya, xa);
    wait_vmcnt<(NS - 2) * PER>();           // the next step is there,
    __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0): all of this one is in registers
    lds_barrier();
    issue(s + NS, st);
    read(after, 0, ya, xa);
    products(yb, xb);
    st = after;
  }
  wait_vmcnt<0>();
  __builtin_amdgcn_s_waitcnt(0xC07F);
  lds_barrier();
  constexpr int SHARE = NS * STAGE / (WM * WN);
  linear_epilogue<OUT, S8OP, RBW, NBW, XT, true, SHARE>(p, acc, m0 + wm * (RBW * 16), n0 + wn * (NBW * 16), lane, ring + wave * SHARE, of_slice);
}

// ---- the large tile: the same step, with loads and fragment reads dealt out among the products, a load per row block (all
// eight at once hold a wave up until the address unit, 64 bytes per clock, has taken the 64 KB of all waves: 8192 x 4096 x
// 4096 215 us, so 210), and the half of the products that loads at raised priority (207).  8192^3 bf16: 735 us, 1.5
// PFLOP/s, the matrix cores busy 78 % of the time at 1.82 GHz, the chip's limit of power (on zeros, without loads, it
// holds 2.42).  One workgroup per CU that goes on to the next tile, whose first steps it loads during the epilogue, takes 780.
template <class T, class OUT, bool XT, bool YT>
__global__ __launch_bounds__(512) void linear_large_kernel(const LinearParams p, int tiles_m, int tiles_n) {
  using E = Elem<T>;
  using AccV = typename E::AccV;
  constexpr bool S8OP = E::kBytes == 1;
  static_assert(!S8OP || (!XT && !YT), "8-bit operands are contiguous along k");
  constexpr int WN = 4, RBW = 8, NBW = 4;      // 2 x 4 waves of 128 x 64
  using OpY = LinearOperand<256, 2, 8, YT, RBW, false>;
  using OpX = LinearOperand<256, 2, 8, XT, NBW, !XT>;
  constexpr int STAGE = (OpY::VECS + OpX::VECS) * 16;
  constexpr int PER = OpY::IP + OpX::IP;
  static_assert(PER == RBW, "a load per row block");
  __shared__ __attribute__((aligned(16))) char ring[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tile_m, tile_n;
  const int of_slice = linear_tile(tiles_m, tiles_n, &tile_m, &tile_n);
  const int64_t m0 = (int64_t)tile_m * 256;
  const int n0 = tile_n * 256;
  OpY y;
  OpX x;
  const LinearSlice slice = linear_slice(p, OpY::BK, of_slice);
  y.begin(wave, lane, p.Y, m0, p.m, p.ldy, p.k, slice.first);
  x.begin(wave, lane, p.X, n0, p.n, p.ldx, p.k, slice.first);
  int y_rd[YT ? RBW : 2], x_rd[XT ? NBW : 2];
  y.offsets(lane, wm, y_rd);
  x.offsets(lane, wn, x_rd);
  AccV acc[RBW][NBW];
#pragma unroll
  for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = AccV{0, 0, 0, 0};
  const uint32_t ring_at = lds_addr(ring);
  auto aim = [&](int s, int stage) __attribute__((always_inline)) {
    const uint32_t st = ring_at + (uint32_t)__builtin_amdgcn_readfirstlane(stage * STAGE);
    y.aim(st, wave, lane, s < slice.steps);
    x.aim(st + OpY::VECS * 16, wave, lane, s < slice.steps);
  };
  auto issue_one = [&](int t) __attribute__((always_inline)) {
    if (t < OpY::IP) y.issue_one(t);
    else x.issue_one(t - OpY::IP);
  };
  v4i ya[RBW], xa[NBW], yb[RBW], xb[NBW];   // the fragments of two halves
  // the products of one half, the reads of the next one (of `stage`) and, with LOADS, those that were aimed in between
  auto half = [&](auto loads, v4i (&yc)[RBW], v4i (&xc)[NBW], int stage, int next, v4i (&yn)[RBW], v4i (&xn)[NBW]) __attribute__((always_inline)) {
    const char *st = ring + stage * STAGE;
#pragma unroll
    for (int rb = 0; rb < RBW; ++rb) {
#pragma unroll
      for (int i = 0; i < RBW + NBW; ++i) {
        if (i * RBW / (RBW + NBW) != rb) continue;
        if (i < NBW) xn[i] = OpX::fragment(st + OpY::VECS * 16, x_rd, next, i);
        else yn[i - NBW] = OpY::fragment(st, y_rd, next, i - NBW);
      }
      if constexpr (decltype(loads)::value) issue_one(rb);
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = E::mfma(xc[nb], yc[rb], acc[rb][nb]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    aim(s, s);
#pragma unroll
    for (int t = 0; t < PER; ++t) issue_one(t);
  }
  wait_vmcnt<PER>();
  lds_barrier();
#pragma unroll
  for (int nb = 0; nb < NBW; ++nb) xa[nb] = OpX::fragment(ring + OpY::VECS * 16, x_rd, 0, nb);
#pragma unroll
  for (int rb = 0; rb < RBW; ++rb) ya[rb] = OpY::fragment(ring, y_rd, 0, rb);
  for (int s = 0; s < slice.steps; ++s) {
    const int st = s & 1;
    half(std::false_type{}, ya, xa, st, 1, yb, xb);
    wait_vmcnt<0>();                        // the next step is there,
    __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0): all of this one is in registers
    lds_barrier();
    __builtin_amdgcn_s_setprio(1);
    aim(s + 2, st);
    half(std::true_type{}, yb, xb, st ^ 1, 0, ya, xa);
    __builtin_amdgcn_s_setprio(0);
  }
  wait_vmcnt<0>();
  __builtin_amdgcn_s_waitcnt(0xC07F);
  lds_barrier();
  constexpr int SHARE = 2 * STAGE / 8;
  linear_epilogue<OUT, S8OP, RBW, NBW, XT, true, SHARE>(p, acc, m0 + wm * (RBW * 16), n0 + wn * (NBW * 16), lane, ring + wave * SHARE, of_slice);
}

// ---- few rows: MB blocks of 16 of them, 16 columns per workgroup, the steps dealt out to its W waves.  What counts is the
// weight, read once from memory: every wave streams its share of 16 weight rows through a ring of its own, no barrier,
// no wait for others; the waves' sums are added up in LDS in wave order.
template <class T, class OUT, int W, int MB, int KS, int NS>
__global__ __launch_bounds__(W * 64) void linear_few_kernel(const LinearParams p) {
  using E = Elem<T>;
  using AccV = typename E::AccV;
  constexpr bool S8OP = E::kBytes == 1;
  using OpY = LinearOperand<MB * 16, KS, 1, false, MB, false>;
  using OpX = LinearOperand<16, KS, 1, false, 1, false>;
  constexpr int STAGE = (OpY::VECS + OpX::VECS) * 16;
  constexpr int L = NS - 1, PER = OpY::IP + OpX::IP;
  static_assert(L * PER < 64 && NS * STAGE >= MB * 1024, "the ring holds a wave's sums");
  __shared__ __attribute__((aligned(16))) char ring[W][NS * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = (int)blockIdx.x * 16;
  OpY y;
  OpX x;
  y.begin(0, lane, p.Y, 0, p.m, p.ldy, p.k, wave);
  x.begin(0, lane, p.X, n0, p.n, p.ldx, p.k, wave);
  int y_rd[KS], x_rd[KS];
  y.offsets(lane, 0, y_rd);
  x.offsets(lane, 0, x_rd);
  const int steps = (int)((p.k + OpY::BK - 1) / OpY::BK), mine = steps > wave ? (steps - wave + W - 1) / W : 0;
  AccV acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = AccV{0, 0, 0, 0};
  const uint32_t ring_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(&ring[wave][0]));
  auto issue = [&](int j, int stage) __attribute__((always_inline)) {
    const uint32_t st = ring_at + (uint32_t)__builtin_amdgcn_readfirstlane(stage * STAGE);
    y.issue_next(st, 0, lane, j < mine);
    x.issue_next(st + OpY::VECS * 16, 0, lane, j < mine);
    y.skip(W - 1);      // (the other waves' steps)
    x.skip(W - 1);
  };
  for (int j = 0; j < L; ++j) issue(j, j);
  int cs = 0, ls = L;
  for (int j = 0; j < mine; ++j) {
    wait_vmcnt<(L - 1) * PER>();
    asm volatile("" ::: "memory");
    const char *st = &ring[wave][cs * STAGE];
    v4i yf[MB][KS], xf[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) xf[k] = OpX::fragment(st + OpY::VECS * 16, x_rd, k, 0);
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int k = 0; k < KS; ++k) yf[b][k] = OpY::fragment(st, y_rd, k, b);
    issue(j + L, ls);
    cs = cs + 1 == NS ? 0 : cs + 1;
    ls = ls + 1 == NS ? 0 : ls + 1;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[b] = E::mfma(xf[k], yf[b][k], acc[b]);
  }
  wait_vmcnt<0>();
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
  // every wave parks its sums in its own ring: [row][column], 16 of those
  const int i = lane & 15, q = lane >> 4;
#pragma unroll
  for (int b = 0; b < MB; ++b) reinterpret_cast<AccV *>(&ring[wave][0])[(b * 16 + i) * 4 + q] = acc[b];
  __syncthreads();
  for (int t = tid; t < MB * 32; t += W * 64) {
    const int m = t >> 1, piece = t & 1, n = n0 + piece * 8;
    if (m >= p.m || n >= p.n) continue;
    const int at = m * 4 + piece * 2;
    AccV a = reinterpret_cast<const AccV *>(&ring[0][0])[at], b = reinterpret_cast<const AccV *>(&ring[0][0])[at + 1];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      a += reinterpret_cast<const AccV *>(&ring[w][0])[at];
      b += reinterpret_cast<const AccV *>(&ring[w][0])[at + 1];
    }
    float v[8], bias[8], scale[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)a[e], v[4 + e] = (float)b[e];
    linear_columns<OUT, S8OP>(p, n, bias, scale);
    linear_finish8<OUT, S8OP, false>(p, m, n, v, bias, scale);
  }
}

// ---- rows as they lie, at any alignment: pieces of 16 bytes go through registers into LDS, SETS steps of them on their way, instead
// of a copy of the operands and a launch for it.  Every load is made on every path (the compiler counts them): behind the end
// of a row its last 16 bytes, which the last step shifts to where they belong, zeros behind them.  Loads at odd addresses bound
// it, a quarter of the rate of aligned ones: 0.45 us a step for the 16 KB of a workgroup, with one step, three or four on the way
// and with steps of 128 k all the same, 0.33 with several workgroups on the CU.  Whole words, put together
// in registers with the one behind them, take longer: 15465 x 1603 -> 64 20.2 us with a load for that word, 19.6 with the next lane's,
// against 16.5.
template <int ROWS, int KS, int WAVES, int SLAB_BLOCKS, bool WIDE_ORDER>
struct AnyOperand : DenseOperand<ROWS, KS, WAVES, false, SLAB_BLOCKS, WIDE_ORDER> {
  using Base = DenseOperand<ROWS, KS, WAVES, false, SLAB_BLOCKS, WIDE_ORDER>;
  const char *row[Base::IP];
  int at[Base::IP];      // byte of the row

  __device__ __forceinline__ void begin(int wave, int lane, const void *ptr, int64_t first, int64_t count, int64_t ld, int step) {
#pragma unroll
    for (int t = 0; t < Base::IP; ++t) {
      const int slot = (wave * Base::IP + t) * 64 + lane;
      const int rho = slot / Base::LPR, c = (slot % Base::LPR) ^ Base::swap_kc(rho);
      const int i = rho & 15, nb = (rho >> 4) % SLAB_BLOCKS, slab = rho / (16 * SLAB_BLOCKS);
      const int64_t r = first + (WIDE_ORDER ? slab * (16 * SLAB_BLOCKS) + (nb >> 1) * 32 + (i >> 2) * 8 + (nb & 1) * 4 + (i & 3) : rho);
      row[t] = reinterpret_cast<const char *>(ptr) + (r < count ? r : count - 1) * ld;      // (rows behind the last are not stored)
      at[t] = step * (Base::BK * 2) + c * 16;
    }
  }
  __device__ __forceinline__ void load(v4i (&to)[Base::IP], int bytes) {
#pragma unroll
    for (int t = 0; t < Base::IP; ++t) {
      to[t] = *reinterpret_cast<const v4i_any1 *>(row[t] + (at[t] < bytes - 16 ? at[t] : bytes - 16));
      at[t] += Base::BK * 2;
    }
  }
  // the pieces of the step `ahead` steps before the next load
  __device__ __forceinline__ void store(char *lds, int wave, int lane, v4i (&from)[Base::IP], bool last, int ahead, int bytes) const {
#pragma unroll
    for (int t = 0; t < Base::IP; ++t) {
      if (last) {
        const int left = bytes - (at[t] - ahead * (Base::BK * 2)), bits = (16 - left) * 8;
        if (left < 16) {
          uint64_t lo = (uint32_t)from[t][0] | (uint64_t)(uint32_t)from[t][1] << 32, hi = (uint32_t)from[t][2] | (uint64_t)(uint32_t)from[t][3] << 32;
          lo = left <= 0 ? 0 : (bits >= 64 ? hi >> (bits - 64) : lo >> bits | hi << (64 - bits));
          hi = left <= 8 ? 0 : hi >> bits;
          from[t] = v4i{(int)(uint32_t)lo, (int)(uint32_t)(lo >> 32), (int)(uint32_t)hi, (int)(uint32_t)(hi >> 32)};
        }
      }
      *reinterpret_cast<v4i *>(lds + ((wave * Base::IP + t) * 64 + lane) * 16) = from[t];
    }
  }
};
template <class T, class OUT, int WM, int WN, int RBW, int NBW, int KS, int SETS>
__global__ __launch_bounds__(WM *WN * 64) void linear_any_kernel(const LinearParams p, int tiles_m, int tiles_n) {
  using E = Elem<T>;
  using AccV = typename E::AccV;
  constexpr int TM = WM * RBW * 16, TN = WN * NBW * 16;
  using OpY = AnyOperand<TM, KS, WM * WN, RBW, false>;
  using OpX = AnyOperand<TN, KS, WM * WN, NBW, true>;
  constexpr int STAGE = (OpY::VECS + OpX::VECS) * 16;
  __shared__ __attribute__((aligned(16))) char ring[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  int tile_m, tile_n;
  const int of_slice = linear_tile(tiles_m, tiles_n, &tile_m, &tile_n);
  const int64_t m0 = (int64_t)tile_m * TM;
  const int n0 = tile_n * TN;
  const LinearSlice slice = linear_slice(p, OpY::BK, of_slice);
  const int bytes = p.row_bytes, final = (bytes + OpY::BK * 2 - 1) / (OpY::BK * 2) - 1 - slice.first;      // the step that ends the rows
  OpY y;
  OpX x;
  y.begin(wave, lane, p.Y, m0, p.m, p.ldy, slice.first);
  x.begin(wave, lane, p.X, n0, p.n, p.ldx, slice.first);
  int y_rd[KS], x_rd[KS];
  y.offsets(lane, wm, y_rd);
  x.offsets(lane, wn, x_rd);
  AccV acc[RBW][NBW];
#pragma unroll
  for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = AccV{0, 0, 0, 0};
  v4i ys[SETS][OpY::IP], xs[SETS][OpX::IP];
#pragma unroll
  for (int j = 0; j < SETS; ++j) {
    y.load(ys[j], bytes);
    x.load(xs[j], bytes);
  }
  for (int s0 = 0; s0 < slice.steps; s0 += SETS) {
#pragma unroll
    for (int j = 0; j < SETS; ++j) {
      const int s = s0 + j;
      if (s >= slice.steps) break;
      // (a stage is written again two steps later: everybody has passed the barrier of the step between, and so read it)
      char *st = ring + (s & 1) * STAGE;
      y.store(st, wave, lane, ys[j], s == final, SETS, bytes);
      x.store(st + OpY::VECS * 16, wave, lane, xs[j], s == final, SETS, bytes);
      y.load(ys[j], bytes);
      x.load(xs[j], bytes);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
      lds_barrier();
      v4i yf[RBW][KS], xf[NBW][KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int nb = 0; nb < NBW; ++nb) xf[nb][k] = OpX::fragment(st + OpY::VECS * 16, x_rd, k, nb);
#pragma unroll
        for (int rb = 0; rb < RBW; ++rb) yf[rb][k] = OpY::fragment(st, y_rd, k, rb);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int rb = 0; rb < RBW; ++rb)
#pragma unroll
          for (int nb = 0; nb < NBW; ++nb) acc[rb][nb] = E::mfma(xf[nb][k], yf[rb][k], acc[rb][nb]);
    }
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  lds_barrier();
  constexpr int SHARE = 2 * STAGE / (WM * WN);
  linear_epilogue<OUT, E::kBytes == 1, RBW, NBW, false, false, SHARE>(p, acc, m0 + wm * (RBW * 16), n0 + wn * (NBW * 16), lane, ring + wave * SHARE, of_slice);
}

// The slices' sums added up, and the epilogue: eight columns of a row by LANES threads, which take every LANES-th slice in
// order and are then added up in order themselves (few outputs and many slices: a chain of loads is LANES times as short)
template <class OUT, bool S8, int LANES>
__global__ __launch_bounds__(256) void linear_join_kernel(const LinearParams p) {
  typedef std::conditional_t<S8, v4i, v4f> V;
  constexpr int ITEMS = 256 / LANES;
  __shared__ V lds[LANES > 1 ? 2 * 256 : 1];
  const int pieces = (p.n + 7) >> 3, item = threadIdx.x % ITEMS, part = threadIdx.x / ITEMS;
  const int64_t i = (int64_t)blockIdx.x * ITEMS + item, all = p.m * pieces;
  const V *at = reinterpret_cast<const V *>(p.partial) + i * 2;
  V a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
  if (i < all) {
#pragma unroll 4
    for (int s = part; s < p.slices; s += LANES) {
      a += at[s * all * 2];
      b += at[s * all * 2 + 1];
    }
  }
  if constexpr (LANES > 1) {
    lds[threadIdx.x * 2] = a;
    lds[threadIdx.x * 2 + 1] = b;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int l = 1; l < LANES; ++l) {
      a += lds[(l * ITEMS + item) * 2];
      b += lds[(l * ITEMS + item) * 2 + 1];
    }
  }
  if (i >= all) return;
  const int64_t m = i / pieces;
  const int n = (int)(i - m * pieces) * 8;
  float v[8], bias[8], scale[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)a[e], v[4 + e] = (float)b[e];
  linear_columns<OUT, S8>(p, n, bias, scale);
  linear_finish8<OUT, S8, false>(p, m, n, v, bias, scale);
}

// Operands whose rows do not lie on 16-byte borders, or end between them: copies whose rows do, zeros behind their
// ends.  thread = 16 bytes of a row; both operands of a product in one launch (none: no rows).
struct LinearRepack {
  struct One {
    void *to;
    const void *from;
    int64_t rows, cols, ld, to_ld;      // elements, to_ld bytes (a multiple of 16)
    int64_t pieces, wgs;
  } of[2];
};
template <int ES>
__global__ __launch_bounds__(256) void linear_repack_kernel(const LinearRepack p) {
  using U = std::conditional_t<ES == 1, uint8_t, uint16_t>;
  using At = std::conditional_t<ES == 1, v4i_any1, v4i_any>;
  constexpr int PER = 16 / ES;
  const bool second = (int64_t)blockIdx.x >= p.of[0].wgs;
  const LinearRepack::One &o = p.of[second];
  const int64_t first = (int64_t)blockIdx.x - (second ? p.of[0].wgs : 0);
  for (int64_t t = first * 256 + threadIdx.x; t < o.rows * o.pieces; t += o.wgs * 256) {
    const int64_t r = t / o.pieces, c = (t - r * o.pieces) * PER;
    const U *src = reinterpret_cast<const U *>(o.from) + r * o.ld + c;
    v4i v;
    if (c + PER <= o.cols) {
      v = *reinterpret_cast<const At *>(src);
    } else {
      U *u = reinterpret_cast<U *>(&v);
#pragma unroll
      for (int e = 0; e < PER; ++e) u[e] = c + e < o.cols ? src[e] : (U)0;
    }
    reinterpret_cast<v4i *>(o.to)[r * (o.to_ld / 16) + c / PER] = v;
  }
}

}  // namespace cummhip
