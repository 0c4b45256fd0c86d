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

// Sum and maximum over the G threads of a row (G = 64, 256 or 1024: waves of a workgroup whose rows are G threads each);
// what a wave has of both goes through LDS.  All threads of the workgroup come here equally often.
template <int G>
__device__ __forceinline__ void row_sum_max(float &sum, float &top, float2 *lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
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

// The whole number next to 127 v / top.  q = v * (127 / top) in 32 bits is within 2^-16 of it (three roundings of at most
// 2^-24 of 127); where a tie may be that near, the two sides of the tie are compared exactly: 254 |v| against (2 n + 1) top, each
// a product of 24 by 9 bits.
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

// G threads per row, P pieces of eight elements each: rows of up to 8 G P elements.  Longer rows (LONG) are read again
// for the second half, from the cache if it holds them.
template <class T, bool NORM, bool CODES, int G, int P, bool LONG>
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
      if (c < k) x[j].load(p.x, row * p.ldx + c, k - c);
      if constexpr (NORM) {
        if (p.residual != nullptr && c < k) r[j].load(p.residual, row * p.ldr + c, k - c);
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
          x[j].store(p.total, row * p.k + c, k - c);
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
        x[j].store(p.out, row * p.k + c, k - c);
      }
    }
  }
}

// A workgroup of 1024 threads takes 1024 / G rows at a time, each thread the same columns of all its rows, so that the
// weight is read once and dw adds up in registers: one row of partial sums per workgroup, added up in order
// (column_sum.h).  All rows' loads of a trip are on their way before its reduction, the next trip's before its use.
template <class T, int G, int P>
__global__ __launch_bounds__(1024) void norm_backward_kernel(const NormGradParams p) {
  __shared__ float2 lds[16];
  __shared__ float sums[G < 1024 ? 8 * G * P : 1];
  constexpr int ROWS = 1024 / G;
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int k = p.k;
  float w[P][8], dw[P][8];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (lane + j * G) * 8;
    Piece<T> t;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[j][e] = dw[j][e] = 0.0f;
    if (c < k) {
      t.load(p.weight, c, k - c);
      t.values(w[j]);
    }
  }
  const float per = 1.0f / (float)k;
  Piece<T> h[P], g[P], s[P];
  float inv = 0.0f;
  const auto fetch = [&](int64_t row) __attribute__((always_inline)) {
    const bool live = row < p.rows;
    inv = live ? p.inv[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (lane + j * G) * 8;
      h[j].raw = g[j].raw = s[j].raw = v4i{0, 0, 0, 0};
      if (c < k && live) {
        h[j].load(p.h, row * p.ldh + c, k - c);
        if (p.grad != nullptr) g[j].load(p.grad, row * p.ldg + c, k - c);
        if (p.grad_total != nullptr) s[j].load(p.grad_total, row * p.ldt + c, k - c);
      }
    }
  };
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  const int64_t stride = (int64_t)gridDim.x * ROWS, trips = (p.rows + stride - 1) / stride;
  fetch(row);
  for (int64_t trip = 0; trip < trips; ++trip, row += stride) {
    float u[P][8], gw[P][8], ds[P][8], dot = 0.0f, none = 0.0f;
    const float i = inv;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      h[j].values(u[j]);
      g[j].values(gw[j]);
      s[j].values(ds[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[j][e] *= i;
        dw[j][e] = __builtin_fmaf(gw[j][e], u[j][e], dw[j][e]);
        gw[j][e] *= w[j][e];
        dot = __builtin_fmaf(gw[j][e], u[j][e], dot);
      }
    }
    const bool live = row < p.rows;
    fetch(row + stride);
    row_sum_max<G>(dot, none, lds);
    const float mean = dot * per;
    if (!live || p.grad_in == nullptr) continue;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (lane + j * G) * 8;
      if (c >= k) continue;
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = __builtin_fmaf(i, gw[j][e] - u[j][e] * mean, ds[j][e]);
      Piece<T> out;
      out.round(d);
      out.store(p.grad_in, row * (int64_t)k + c, k - c);
    }
  }
  if (p.partial == nullptr) return;
  if constexpr (ROWS > 1) {      // the row groups' sums, in their order
    for (int r = 0; r < ROWS; ++r) {
      if (group == r) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          float *at = sums + (lane + j * G) * 8;
#pragma unroll
          for (int e = 0; e < 8; ++e) at[e] = r == 0 ? dw[j][e] : at[e] + dw[j][e];
        }
      }
      __syncthreads();
    }
    float *to = p.partial + (int64_t)blockIdx.x * p.pitch;
    for (int c = threadIdx.x; c < p.pitch; c += 1024) to[c] = c < 8 * G * P ? sums[c] : 0.0f;
  } else {
    float *to = p.partial + (int64_t)blockIdx.x * p.pitch;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (lane + j * G) * 8;
      if (c >= p.pitch) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) to[c + e] = dw[j][e];
    }
  }
}

// Rows longer than the registers of a workgroup hold: one row per workgroup and trip, read twice.  dw of a
// workgroup adds up in its row of the partial sums.
template <class T>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const NormGradParams p) {
  __shared__ float2 lds[16];
  const int k = p.k, lane = threadIdx.x;
  float *mine = p.partial != nullptr ? p.partial + (int64_t)blockIdx.x * p.pitch : nullptr;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const bool first_row = row == blockIdx.x;
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
        h.values(u);
        g.values(gv);
        w.values(wv);
        if (pass == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u[e] *= i;
            dot = __builtin_fmaf(gv[e] * wv[e], u[e], dot);
            if (mine != nullptr) mine[c + e] = __builtin_fmaf(gv[e], u[e], first_row ? 0.0f : mine[c + e]);
          }
        } else if (p.grad_in != nullptr) {
          if (p.grad_total != nullptr) s.load(p.grad_total, row * p.ldt + c, k - c);
          s.values(sv);
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
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= linear_act_slope(zf[e], p.act, p.slope);
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
  const float total = column_final_sum(partial, pitch, 0, blocks, blockIdx.x);
  const int c = blockIdx.x * 16 + threadIdx.x;
  if (threadIdx.x < 16 && c < n) reinterpret_cast<uint16_t *>(dst)[c] = Elem<T>::from_float(total);
}

constexpr size_t kStreamBytes = (size_t)64 << 20;      // operands that are read past the caches

template <class T, bool NORM, bool CODES, int G, int P, bool LONG = false>
hipError_t norm_as(const NormParams &p, hipStream_t s) {
  constexpr int ROWS = G < 256 ? 256 / G : 1;
  const int64_t wgs = (p.rows + ROWS - 1) / ROWS;
  const int64_t wide = std::min<int64_t>(wgs, 1 << 21);      // (a launch has fewer than 2^32 threads along a side)
  hipLaunchKernelGGL((norm_kernel<T, NORM, CODES, G, P, LONG>), dim3((unsigned)wide, (unsigned)((wgs + wide - 1) / wide)), dim3(G < 256 ? 256 : G), 0, s, p);
  return hipGetLastError();
}
template <class T, bool NORM, bool CODES>
hipError_t norm_of(const NormParams &p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  if (p.k <= 512) return norm_as<T, NORM, CODES, 64, 1>(p, s);
  if (p.k <= 1024) return norm_as<T, NORM, CODES, 64, 2>(p, s);
  if (p.k <= 2048) return norm_as<T, NORM, CODES, 256, 1>(p, s);
  if (p.k <= 4096) return norm_as<T, NORM, CODES, 256, 2>(p, s);
  if (p.k <= 8192) return norm_as<T, NORM, CODES, 256, 4>(p, s);
  if (p.k <= 16384) return norm_as<T, NORM, CODES, 1024, 2>(p, s);
  if (p.k <= 32768) return norm_as<T, NORM, CODES, 1024, 4>(p, s);
  return norm_as<T, NORM, CODES, 1024, 4, true>(p, s);
}

template <class T>
hipError_t norm_backward_of(const NormGradParams &p, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks);
  if (p.k <= 512) hipLaunchKernelGGL((norm_backward_kernel<T, 64, 1>), grid, dim3(1024), 0, s, p);
  else if (p.k <= 1024) hipLaunchKernelGGL((norm_backward_kernel<T, 64, 2>), grid, dim3(1024), 0, s, p);
  else if (p.k <= 2048) hipLaunchKernelGGL((norm_backward_kernel<T, 256, 1>), grid, dim3(1024), 0, s, p);
  else if (p.k <= 4096) hipLaunchKernelGGL((norm_backward_kernel<T, 256, 2>), grid, dim3(1024), 0, s, p);
  else if (p.k <= 8192) hipLaunchKernelGGL((norm_backward_kernel<T, 1024, 1>), grid, dim3(1024), 0, s, p);
  else if (p.k <= 16384) hipLaunchKernelGGL((norm_backward_kernel<T, 1024, 2>), grid, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL(norm_backward_long_kernel<T>, grid, dim3(1024), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.partial == nullptr) return e;
  hipLaunchKernelGGL(rows_sum_kernel<T>, dim3((unsigned)(p.pitch / 16)), dim3(256), 0, s, p.partial, p.blocks, p.pitch, p.grad_weight, p.k);
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

// Workgroups of the backward pass: two rounds of the device's 2 x 256 resident ones at most, a row group each at least
int norm_backward_blocks(int64_t rows, int k) {
  const int at_once = k <= 1024 ? 16 : (k <= 4096 ? 4 : 1);
  const int64_t wgs = (rows + at_once - 1) / at_once;
  return (int)(wgs < 512 ? (wgs > 0 ? wgs : 1) : 512);
}
hipError_t launch_norm_backward(const NormGradParams &p, bool bf16, hipStream_t s) {
  return bf16 ? norm_backward_of<BF16>(p, s) : norm_backward_of<F16>(p, s);
}

// A strip is 32 pieces of eight columns, fewer for narrow rows; blocks of rows so that there are some 1024 workgroups, of at
// least one trip of 4 rows per thread
void linear_gate_shape(int64_t rows, int n, int *shift, int *strips, int *blocks, int64_t *per) {
  const int pieces = (n + 7) / 8;
  *shift = 0;
  while (*shift < 5 && (1 << *shift) < pieces) ++*shift;
  *strips = (pieces + (1 << *shift) - 1) >> *shift;
  const int64_t trip = 4 * (256 >> *shift);
  int64_t want = 1024 / *strips;
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
  if (bf16) hipLaunchKernelGGL(rows_sum_kernel<BF16>, dim3((unsigned)(p.pitch / 16)), dim3(256), 0, s, p.partial, blocks, p.pitch, grad_bias, p.n);
  else hipLaunchKernelGGL(rows_sum_kernel<F16>, dim3((unsigned)(p.pitch / 16)), dim3(256), 0, s, p.partial, blocks, p.pitch, grad_bias, p.n);
  return hipGetLastError();
}

}  // namespace cummhip
