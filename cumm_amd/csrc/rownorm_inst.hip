// Root-mean-square norm of rows with the residual's addition, its gradients, and rows in 8 bits with a scale each:
//
//   norm      h = round(x + r)  (or x);  i = 1 / sqrt(mean of h^2 + eps);  y = round(h i w)
//   in 8 bits v = h w, top = largest |v| of the row;  code = whole number next to 127 v / top, ties to even;
//             scale = i top / 127        (code * scale is y in 8 bits; without the norm: i = w = 1)
//   backward  u = h i, g = gradient of y, s = gradient of h as it is used elsewhere:
//             dh = i (g w - u mean of g w u) + s  (it is the gradient of x and of r);  dw = sum over rows of g u
//
// The sum is rounded to the type before the norm: that is what is stored, what the next layer adds to, and what the
// backward pass has.  Statistics and products are 32 bits; every result is rounded once.  The code of an element depends on
// no order of a sum: v is exact in 32 bits (two-byte factors; a 32-bit row has no factor), and so is the comparison that
// decides where the 32-bit quotient lies next to a tie.
//
// All of it is bound by memory: a row is read once, held in registers, and both sums of it - of the squares
// and the maximum - go through one reduction.
#include <algorithm>

#include "column_sum.h"
#include "layers.h"
#include "linear.h"
#include "rows.h"

namespace cummhip {

namespace {

// Sum and maximum over the G threads of a row: lanes of a wave (G up to 64; narrow rows, as voxels have them, are several
// to a wave), or whole waves of a workgroup, which exchange what they have through LDS.  All threads of the workgroup
// come here equally often.
template <int G>
__device__ __forceinline__ void row_sum_max(float &sum, float &top, float2 *lds) {
#pragma unroll
  for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, 64);
    const float other = __shfl_xor(top, off, 64);
    top = other > top || other != other ? other : top;      // (NaN stays)
  }
  if constexpr (G > 64) {
    constexpr int WAVES = G / 64;
    const int wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
    if ((threadIdx.x & 63) == 0) lds[wave] = make_float2(sum, top);
    __syncthreads();
    sum = 0.0f;
    top = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 v = lds[first + w];
      sum += v.x;
      top = v.y > top || v.y != v.y ? v.y : top;
    }
    __syncthreads();
  }
}

// The whole number next to 127 v / top.  q = v * (127 / top) in 32 bits is within 1.52e-5 of it: two roundings, of the quotient and of the
// product, of at most 2^-24 of 127 each (the lift below is a power of two).  Where a tie is nearer than twice that, the two sides of the
// tie are compared exactly: 254 |v| against (2 n + 1) top, each a product of 24 by 9 bits.
__device__ __forceinline__ int code_of(float v, float inv, double top) {
  const float q = v * inv, r = __builtin_rintf(q);
  int code = (int)r;
  if (__builtin_expect(__builtin_fabsf(__builtin_fabsf(q - r) - 0.5f) < 3.1e-5f, 0)) {
    const float a = __builtin_fabsf(q);
    const int n = (int)a;                          // the tie next to it is n + 1/2
    const double left = 254.0 * (double)__builtin_fabsf(v), right = (double)(2 * n + 1) * top;
    const int near = left > right ? n + 1 : (left < right ? n : n + (n & 1));
    code = v < 0.0f ? -near : near;
  }
  return code;
}

struct RowScale {
  float inv;         // 127 / top of the scaled row
  double top;
  float lift;        // 1, or a power of two that lifts a row of tiny numbers to where 127 / top is finite
  bool codes;        // there are codes: a row of zeros, or with an infinity or NaN in it, has none
};
__device__ __forceinline__ RowScale row_scale(float top) {
  RowScale s;
  s.lift = top < 0x1p-96f ? 0x1p64f : 1.0f;
  const float lifted = top * s.lift;
  s.codes = lifted > 0.0f && lifted < __builtin_inff();
  s.inv = s.codes ? 127.0f / lifted : 0.0f;
  s.top = (double)lifted;
  return s;
}

template <int P>
__device__ __forceinline__ void write_codes(int8_t *codes, int first, int k, int lane, int G, const float (&v)[P][8], float top) {
  const RowScale s = row_scale(top);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = first + (lane + j * G) * 8;
    if (c >= k) continue;
    int b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = s.codes ? code_of(v[j][e] * s.lift, s.inv, s.top) : 0;
    const v2i_any two = {pack4_bytes(b[0], b[1], b[2], b[3]), pack4_bytes(b[4], b[5], b[6], b[7])};
    int8_t *dst = codes + c;
    if (c + 8 <= k) {
      *reinterpret_cast<v2i_any *>(dst) = two;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < k) dst[e] = (int8_t)b[e];
    }
  }
}

// Operands of this size are read, and results written, past the caches: 16384 rows of 4096 with a residual 96 -> 87 us, 8191 of
// 5120 to 8 bits 58 -> 51, 8192 of 8192 to 8 bits without a norm 38 -> 35.  What is smaller the next launch finds there.
constexpr size_t kStreamBytes = (size_t)64 << 20;

// G threads per row, P pieces of eight elements each: rows of up to 8 G P elements.  Longer rows (LONG) are read again
// for the second half, from the cache if it holds them.
template <class T, bool NORM, bool CODES, int G, int P, bool LONG, bool NT>
__global__ __launch_bounds__(G < 256 ? 256 : G) void norm_kernel(const NormParams p) {
  __shared__ float2 lds[16];
  constexpr int ROWS = G < 256 ? 256 / G : 1;
  const int lane = threadIdx.x % G;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / G;
  const bool live = row < p.rows;
  const int k = live ? p.k : 0;
  const int trips = LONG ? (p.k + 8 * G * P - 1) / (8 * G * P) : 1;
  float sum = 0.0f, top = 0.0f;
  Piece<T> x[P];
  float v[P][8];
  for (int trip = 0; trip < trips; ++trip) {
    const int first = trip * (8 * G * P);
    Piece<T> r[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = first + (lane + j * G) * 8;
      if (c < k) x[j].template load<NT>(p.x, row * p.ldx + c, k - c);
      if constexpr (NORM) {
        if (p.residual != nullptr && c < k) r[j].template load<NT>(p.residual, row * p.ldr + c, k - c);
      }
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = first + (lane + j * G) * 8;
      if (c >= k) continue;
      float h[8];
      x[j].values(h);
      if constexpr (NORM) {
        if (p.residual != nullptr) {
          float f[8];
          r[j].values(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] += f[e];
          x[j].round(h);
          x[j].template store<NT>(p.total, row * p.k + c, k - c);
          x[j].values(h);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(h[e], h[e], sum);
      }
      if constexpr (CODES) {
        if constexpr (NORM) {
          Piece<T> w;
          float f[8];
          w.load(p.weight, c, k - c);
          w.values(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[j][e] = h[e];
          const float a = __builtin_fabsf(h[e]);
          top = a > top || a != a ? a : top;
        }
      }
    }
  }
  row_sum_max<G>(sum, top, lds);
  float inv = 1.0f;
  if constexpr (NORM) inv = 1.0f / __builtin_sqrtf(sum / (float)p.k + p.eps);
  if (!live) return;
  if (lane == 0) {
    if constexpr (NORM) {
      if (p.inv != nullptr) p.inv[row] = inv;
    }
    if constexpr (CODES) p.scale[row] = inv * (top / 127.0f);
  }
  for (int trip = 0; trip < trips; ++trip) {
    const int first = trip * (8 * G * P);
    if constexpr (LONG) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c = first + (lane + j * G) * 8;
        if (c >= k) continue;
        if (NORM && p.residual != nullptr) x[j].load(p.total, row * p.k + c, k - c);      // (this thread wrote it)
        else x[j].load(p.x, row * p.ldx + c, k - c);
        x[j].values(v[j]);
        if constexpr (NORM && CODES) {
          Piece<T> w;
          float f[8];
          w.load(p.weight, c, k - c);
          w.values(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] *= f[e];
        }
      }
    }
    if constexpr (CODES) {
      write_codes<P>(p.codes + row * p.k, first, k, lane, G, v, top);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c = first + (lane + j * G) * 8;
        if (c >= k) continue;
        Piece<T> w;
        float f[8], h[8];
        w.load(p.weight, c, k - c);
        w.values(f);
        x[j].values(h);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = h[e] * inv * f[e];
        x[j].round(h);
        x[j].template store<NT>(p.out, row * p.k + c, k - c);
      }
    }
  }
}

// A workgroup of 1024 threads takes 1024 / G rows at a time, each thread the same columns of all its rows, so that the
// weight is read once and dw adds up in registers: one row of partial sums per workgroup, added up in order
// (column_sum.h).  The rows of a trip stay as they lie in memory - their values are worked out twice, before and after the
// reduction - so that those of the next one can be on their way (AHEAD) in the 128 registers that a thread has: kept as
// values, 8192 rows of 4096 spill and take 172 us.
template <class T, int G, int P, bool AHEAD, bool NT>
__global__ __launch_bounds__(1024) void norm_backward_kernel(const NormGradParams p) {
  constexpr int ROWS = 1024 / G, WIDTH = 8 * G * P;
  constexpr int PARTS = ROWS < 16 ? ROWS : 16;      // sums of a column that meet in LDS: of row groups, or of waves
  __shared__ float2 lds[16];
  __shared__ float sums[PARTS > 1 ? PARTS * WIDTH : 1];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int k = p.k;
  Piece<T> w[P];
  float dw[P][8];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (lane + j * G) * 8;
    w[j].raw = v4i{0, 0, 0, 0};
    if (c < k) w[j].load(p.weight, c, k - c);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = 0.0f;
  }
  const float per = 1.0f / (float)k;
  struct Row {
    Piece<T> h[P], g[P], s[P];
    float inv;
  };
  const auto fetch = [&](Row &r, int64_t row) __attribute__((always_inline)) {
    const bool live = row < p.rows;
    r.inv = live ? p.inv[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (lane + j * G) * 8;
      r.h[j].raw = r.g[j].raw = r.s[j].raw = v4i{0, 0, 0, 0};
      if (c < k && live) {
        r.h[j].template load<NT>(p.h, row * p.ldh + c, k - c);
        if (p.grad != nullptr) r.g[j].template load<NT>(p.grad, row * p.ldg + c, k - c);
        if (p.grad_total != nullptr) r.s[j].template load<NT>(p.grad_total, row * p.ldt + c, k - c);
      }
    }
  };
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  const int64_t stride = (int64_t)gridDim.x * ROWS, trips = (p.rows + stride - 1) / stride;
  Row now, next;
  fetch(now, row);
  for (int64_t trip = 0; trip < trips; ++trip, row += stride) {
    if constexpr (AHEAD) fetch(next, row + stride);
    float dot = 0.0f, none = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float u[8], g[8], f[8];
      now.h[j].values(u);
      now.g[j].values(g);
      w[j].values(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] *= now.inv;
        dw[j][e] = __builtin_fmaf(g[e], u[e], dw[j][e]);
        dot = __builtin_fmaf(g[e] * f[e], u[e], dot);
      }
    }
    row_sum_max<G>(dot, none, lds);
    const float mean = dot * per;
    if (row < p.rows && p.grad_in != nullptr) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c = (lane + j * G) * 8;
        if (c >= k) continue;
        float u[8], g[8], f[8], d[8];
        now.h[j].values(u);
        now.g[j].values(g);
        now.s[j].values(d);
        w[j].values(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = __builtin_fmaf(now.inv, g[e] * f[e] - u[e] * now.inv * mean, d[e]);
        Piece<T> out;
        out.round(d);
        out.template store<NT>(p.grad_in, row * (int64_t)k + c, k - c);
      }
    }
    if constexpr (AHEAD) now = next;
    else fetch(now, row + stride);
  }
  if (p.partial == nullptr) return;
  float *to = p.partial + (int64_t)blockIdx.x * p.pitch;
  if constexpr (PARTS > 1) {
    // the rows that share a wave, then the waves' or groups' sums in their order
#pragma unroll
    for (int off = 32; off >= G; off >>= 1)
#pragma unroll
      for (int j = 0; j < P; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[j][e] += __shfl_xor(dw[j][e], off, 64);
    const int part = G < 64 ? threadIdx.x >> 6 : group;
    if (G >= 64 || (threadIdx.x & 63) < G) {
#pragma unroll
      for (int j = 0; j < P; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[part * WIDTH + (lane + j * G) * 8 + e] = dw[j][e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.pitch; c += 1024) {
      float t = 0.0f;
      if (c < WIDTH) {
#pragma unroll
        for (int r = 0; r < PARTS; ++r) t += sums[r * WIDTH + c];
      }
      to[c] = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (lane + j * G) * 8;
      if (c >= p.pitch) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) to[c + e] = dw[j][e];
    }
  }
}

// Rows longer than the registers of a workgroup hold: one row per workgroup and trip, read twice.  dw of a workgroup adds
// up in LDS, [element of a piece][piece], or, of the longest rows, in its row of the partial sums.
constexpr int kLongInLds = 32768;
template <class T, bool IN_LDS>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const NormGradParams p) {
  __shared__ float2 lds[16];
  __shared__ float sums[IN_LDS ? kLongInLds : 1];
  const int k = p.k, lane = threadIdx.x;
  float *mine = p.partial != nullptr ? p.partial + (int64_t)blockIdx.x * p.pitch : nullptr;
  const auto at = [&](int c, int e) -> float & { return IN_LDS ? sums[e * (kLongInLds / 8) + (c >> 3)] : mine[c + e]; };
  if (mine != nullptr) {
    for (int c = lane * 8; c < p.pitch; c += 8192)      // (each thread its own columns throughout)
#pragma unroll
      for (int e = 0; e < 8; ++e) at(c, e) = 0.0f;
  }
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float i = p.inv[row];
    float dot = 0.0f, none = 0.0f, mean = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int c = lane * 8; c < k; c += 8192) {
        Piece<T> h, g, s, w;
        float u[8], gv[8], sv[8], wv[8];
        h.load(p.h, row * p.ldh + c, k - c);
        w.load(p.weight, c, k - c);
        g.raw = s.raw = v4i{0, 0, 0, 0};
        if (p.grad != nullptr) g.load(p.grad, row * p.ldg + c, k - c);
        if (pass == 1 && p.grad_total != nullptr) s.load(p.grad_total, row * p.ldt + c, k - c);
        h.values(u);
        g.values(gv);
        w.values(wv);
        s.values(sv);
        if (pass == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u[e] *= i;
            dot = __builtin_fmaf(gv[e] * wv[e], u[e], dot);
            if (mine != nullptr) at(c, e) = __builtin_fmaf(gv[e], u[e], at(c, e));
          }
        } else if (p.grad_in != nullptr) {
          float d[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = __builtin_fmaf(i, gv[e] * wv[e] - u[e] * i * mean, sv[e]);
          Piece<T> out;
          out.round(d);
          out.store(p.grad_in, row * (int64_t)k + c, k - c);
        }
      }
      if (pass == 0) {
        row_sum_max<1024>(dot, none, lds);
        mean = dot / (float)k;
      }
    }
  }
  if (IN_LDS && mine != nullptr) {
    for (int c = lane * 8; c < p.pitch; c += 8192)
#pragma unroll
      for (int e = 0; e < 8; ++e) mine[c + e] = at(c, e);
  }
}

// Gradient through the activation and column sums of it: dz = g act'(z), sums of dz before it is rounded.  A workgroup
// takes a strip of up to 256 columns (32 pieces) of a block of rows, 256 / pieces rows at a time; its sums go to a row
// of partial sums, added up in the order of the blocks.
template <class T, bool NT>
__global__ __launch_bounds__(256) void linear_gate_kernel(const LinearGateParams p) {
  __shared__ float lds[256][9];
  const int pieces = 1 << p.shift, lanes = 256 >> p.shift;
  const int piece = threadIdx.x & (pieces - 1), lane_row = threadIdx.x >> p.shift;
  const int c = ((int)blockIdx.x * pieces + piece) * 8, count = p.n - c;
  const int64_t r0 = (int64_t)blockIdx.y * p.rows_per_block, end = r0 + p.rows_per_block, r1 = end < p.rows ? end : p.rows;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  constexpr int BATCH = 4;
  for (int64_t r = r0 + lane_row; r < r1; r += BATCH * lanes) {
    Piece<T> g[BATCH], z[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int64_t at = r + b * lanes;
      g[b].raw = z[b].raw = v4i{0, 0, 0, 0};
      if (at < r1 && count > 0) {
        g[b].template load<NT>(p.grad, at * p.ldg + c, count);
        if (p.pre != nullptr) z[b].template load<NT>(p.pre, at * p.ldp + c, count);
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int64_t at = r + b * lanes;
      if (at >= r1) continue;
      float f[8], zf[8];
      g[b].values(f);
      z[b].values(zf);
      if (p.pre != nullptr) {
        linear_act_slopes(f, v4f{zf[0], zf[1], zf[2], zf[3]}, v4f{zf[4], zf[5], zf[6], zf[7]}, p.act, p.slope);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += f[e];      // (zeros behind the end: the slope there is finite)
      if (p.dz != nullptr && c < p.ldz) {      // (whole pieces: zeros behind the end of a row)
        Piece<T> out;
        out.round(f);
        out.store(p.dz, at * p.dz_pitch + c, 8);
      }
    }
  }
  if (p.partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) lds[threadIdx.x][e] = sum[e];
  __syncthreads();
  if (lane_row == 0 && c < p.pitch) {
    for (int l = 1; l < lanes; ++l)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += lds[(l << p.shift) + piece][e];
    float *to = p.partial + (int64_t)blockIdx.y * p.pitch + c;
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = sum[e];
  }
}

// partial sums [blocks][pitch] to dst[n], pitch a multiple of 16
template <class T>
__global__ __launch_bounds__(256) void rows_sum_kernel(const float *partial, int blocks, int pitch, void *dst, int n) {
  const int group = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  if (group * 16 >= n) return;
  const float total = column_final_sum(partial, pitch, 0, blocks, group);
  const int c = group * 16 + threadIdx.x;
  if (threadIdx.x < 16 && c < n) reinterpret_cast<uint16_t *>(dst)[c] = Elem<T>::from_float(total);
}

// workgroups of 256 threads for `groups` of 16 columns (a launch has fewer than 2^32 threads along a side)
dim3 rows_sum_grid(int pitch) {
  const int64_t groups = pitch / 16, wide = std::min<int64_t>(groups, 1 << 20);
  return dim3((unsigned)wide, (unsigned)((groups + wide - 1) / wide));
}

template <class T, bool NORM, bool CODES, int G, int P, bool LONG = false>
hipError_t norm_as(const NormParams &p, hipStream_t s) {
  constexpr int ROWS = G < 256 ? 256 / G : 1;
  const int64_t wgs = (p.rows + ROWS - 1) / ROWS;
  const int64_t wide = std::min<int64_t>(wgs, 1 << 21);      // (a launch has fewer than 2^32 threads along a side)
  const dim3 grid((unsigned)wide, (unsigned)((wgs + wide - 1) / wide)), block(G < 256 ? 256 : G);
  if (!LONG && (size_t)p.rows * (size_t)p.k * Elem<T>::kBytes >= kStreamBytes) hipLaunchKernelGGL((norm_kernel<T, NORM, CODES, G, P, LONG, !LONG>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((norm_kernel<T, NORM, CODES, G, P, LONG, false>), grid, block, 0, s, p);
  return hipGetLastError();
}
// Two pieces a thread throughout, for the loads that it has on their way (20000 rows of 1500 with a residual 54 us with one piece
// and 256 threads, 45 with two and 128), as many threads as that takes; four where a row is quantised alone, which is half
// the loads (8192 rows of 8192 40 us with two, 36 with four), and in rows above 8192, where whole workgroups wait for
// each other at the reduction (4000 of 16384 to 8 bits 46 us with 1024 threads, 37 with 512).  Rows of up to 512 share waves
// (30000 of 64 12.6 us with a wave each, 6.4 with eight threads).
template <class T, bool NORM, bool CODES>
hipError_t norm_of(const NormParams &p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  if (p.k <= 64) return norm_as<T, NORM, CODES, 8, 1>(p, s);
  if (p.k <= 128) return norm_as<T, NORM, CODES, 8, 2>(p, s);
  if (p.k <= 256) return norm_as<T, NORM, CODES, 16, 2>(p, s);
  if (p.k <= 512) return norm_as<T, NORM, CODES, 32, 2>(p, s);
  if (p.k <= 1024) return norm_as<T, NORM, CODES, 64, 2>(p, s);
  if (p.k <= 2048) return norm_as<T, NORM, CODES, 128, 2>(p, s);
  if (p.k <= 4096) return norm_as<T, NORM, CODES, 256, 2>(p, s);
  if (p.k <= 8192) return NORM ? norm_as<T, NORM, CODES, 512, 2>(p, s) : norm_as<T, NORM, CODES, 256, 4>(p, s);
  if (p.k <= 16384) return norm_as<T, NORM, CODES, 512, 4>(p, s);
  if (p.k <= 32768) return norm_as<T, NORM, CODES, 1024, 4>(p, s);
  return norm_as<T, NORM, CODES, 1024, 4, true>(p, s);
}

template <class T>
hipError_t norm_backward_of(const NormGradParams &p, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks);
  const bool stream = (size_t)p.rows * (size_t)p.k * 2 >= kStreamBytes;
  const auto launch = [&](auto past, auto kept) {
    if (stream) hipLaunchKernelGGL(past, grid, dim3(1024), 0, s, p);
    else hipLaunchKernelGGL(kept, grid, dim3(1024), 0, s, p);
  };
#define CUMM_NORM(G, P, AHEAD) launch(norm_backward_kernel<T, G, P, AHEAD, true>, norm_backward_kernel<T, G, P, AHEAD, false>)
  if (p.k <= 64) CUMM_NORM(8, 1, true);
  else if (p.k <= 128) CUMM_NORM(16, 1, true);
  else if (p.k <= 256) CUMM_NORM(32, 1, true);
  else if (p.k <= 512) CUMM_NORM(64, 1, true);
  else if (p.k <= 1024) CUMM_NORM(128, 1, true);
  else if (p.k <= 2048) CUMM_NORM(256, 1, true);
  else if (p.k <= 4096) CUMM_NORM(512, 1, true);
  else if (p.k <= 8192) CUMM_NORM(1024, 1, true);
  else if (p.k <= 16384) CUMM_NORM(1024, 2, false);      // (two rows of them do not fit the registers)
#undef CUMM_NORM
  else if (p.k <= kLongInLds) hipLaunchKernelGGL((norm_backward_long_kernel<T, true>), grid, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL((norm_backward_long_kernel<T, false>), grid, dim3(1024), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.partial == nullptr) return e;
  hipLaunchKernelGGL(rows_sum_kernel<T>, rows_sum_grid(p.pitch), dim3(256), 0, s, p.partial, p.blocks, p.pitch, p.grad_weight, p.k);
  return hipGetLastError();
}

__global__ __launch_bounds__(256) void rows_zero_kernel(uint16_t *dst, int64_t elements) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elements; i += (int64_t)gridDim.x * 256) dst[i] = 0;
}

}  // namespace

hipError_t launch_rows_zero(void *dst, int64_t elements, hipStream_t s) {
  if (elements == 0) return hipSuccess;
  const int64_t wgs = std::min<int64_t>((elements + 255) / 256, 4096);
  hipLaunchKernelGGL(rows_zero_kernel, dim3((unsigned)wgs), dim3(256), 0, s, reinterpret_cast<uint16_t *>(dst), elements);
  return hipGetLastError();
}

hipError_t launch_norm(const NormParams &p, int dtype, hipStream_t s) {
  const bool norm = p.weight != nullptr, codes = p.codes != nullptr;
  if (dtype == 0) return codes && !norm ? norm_of<F32, false, true>(p, s) : hipErrorInvalidValue;
  if (dtype == 7) return norm ? (codes ? norm_of<F16, true, true>(p, s) : norm_of<F16, true, false>(p, s)) : norm_of<F16, false, true>(p, s);
  return norm ? (codes ? norm_of<BF16, true, true>(p, s) : norm_of<BF16, true, false>(p, s)) : norm_of<BF16, false, true>(p, s);
}

// Workgroups of the backward pass: one per CU, which is what its registers allow (8192 rows of 4096 52 us, with two 57), a row
// group each at least
constexpr int kNormBlocks = 256;
int norm_backward_blocks(int64_t rows, int k) {
  int at_once = 128;      // rows: 1024 threads of eight columns each
  while (at_once > 1 && k > 8192 / at_once) at_once /= 2;
  const int64_t wgs = (rows + at_once - 1) / at_once;
  return (int)(wgs < kNormBlocks ? (wgs > 0 ? wgs : 1) : kNormBlocks);
}
hipError_t launch_norm_backward(const NormGradParams &p, bool bf16, hipStream_t s) {
  return bf16 ? norm_backward_of<BF16>(p, s) : norm_backward_of<F16>(p, s);
}

// A strip is 32 pieces of eight columns, fewer for narrow rows; blocks of rows so that there are some 1024 workgroups, of at
// least one trip of 4 rows per thread; 4096 of wide rows, whose blocks leave fewer sums each (dz and sums of 8192 x 4096 with the rest of
// a pass 67 us, so 58; 120000 x 256 58.6, with 4096 62.3)
void linear_gate_shape(int64_t rows, int n, int *shift, int *strips, int *blocks, int64_t *per) {
  const int pieces = (n + 7) / 8;
  *shift = 0;
  while (*shift < 5 && (1 << *shift) < pieces) ++*shift;
  *strips = (pieces + (1 << *shift) - 1) >> *shift;
  const int64_t trip = 4 * (256 >> *shift);
  int64_t want = (*strips >= 8 ? 4096 : 1024) / *strips;
  if (want < 1) want = 1;
  int64_t rows_each = (rows + want - 1) / want;
  rows_each = (rows_each + trip - 1) / trip * trip;
  if (rows_each < trip) rows_each = trip;
  *per = rows_each;
  *blocks = (int)((rows + rows_each - 1) / rows_each);
  if (*blocks < 1) *blocks = 1;
}
hipError_t launch_linear_gate(LinearGateParams p, int64_t dz_pitch, void *grad_bias, bool bf16, hipStream_t s) {
  p.dz_pitch = dz_pitch;
  int strips, blocks;
  linear_gate_shape(p.rows, p.n, &p.shift, &strips, &blocks, &p.rows_per_block);
  const dim3 grid((unsigned)strips, (unsigned)blocks);
  const bool stream = (size_t)p.rows * (size_t)p.n * 2 >= kStreamBytes;
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p); };
  if (bf16) stream ? launch(linear_gate_kernel<BF16, true>) : launch(linear_gate_kernel<BF16, false>);
  else stream ? launch(linear_gate_kernel<F16, true>) : launch(linear_gate_kernel<F16, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.partial == nullptr) return e;
  if (bf16) hipLaunchKernelGGL(rows_sum_kernel<BF16>, rows_sum_grid(p.pitch), dim3(256), 0, s, p.partial, blocks, p.pitch, grad_bias, p.n);
  else hipLaunchKernelGGL(rows_sum_kernel<F16>, rows_sum_grid(p.pitch), dim3(256), 0, s, p.partial, blocks, p.pitch, grad_bias, p.n);
  return hipGetLastError();
}

}  // namespace cummhip
