// The backward pass of a layer with few channels on both sides, in one pass over its rows:
//     z = x W^T + b (f32, worked out again: the forward pass writes nothing for it),  dz = grad act'(z) (rounded for the products),
//       or, of an activation with a kink, whose side the forward pass leaves as a bit, dz = grad or slope * grad,
//     grad_x = dz W,  grad_W = sum of dz^T x,  grad_b = sum of dz.
// Three reads and writes of a row (x, grad, grad_x) are all the memory traffic; apart, dz is written and read twice, z written
// and read, x read again.  A wave takes 16 rows through both products in registers: with the weight's rows (columns) as the
// first operand, in the order that gives a lane 8 consecutive channels of every two blocks, a lane holds row lane & 15, channels 8 q ..
// of each 32 (q = lane >> 4) of z as it does of x and grad in memory (16-byte accesses), and dz as it stands is the second operand of the
// product with W.  grad_W contracts over rows: dz and x go through LDS, where the transposing read turns them, and the eight waves
// share its blocks.  The weight lies in LDS as the fragments of both products.  A workgroup goes through its rows with the next
// ones on their way, and leaves one set of sums; they are added in the workgroups' order (the same bits in every run).
// dz is rounded to the operands' type for the matrix instructions, as it is where it is stored between launches; grad_b sums it
// unrounded.
// Measured with all gradients, the launch that adds up the sums (3 - 11 us) not counted: 119985 rows, 64 -> 128 channels, f16, ReLU 22 us (with z worked out
// again 30); 1 M rows, 64 -> 64 80 (4.9 TB/s of what it moves), 128 -> 128 182 (4.3); 1000 rows 10.  With gelu 120 k rows take 32, 1 M of 128 -> 128
// 230: 25 instructions an element, which the loads do not hide.  The gate and two products that read a stored z take 51, 171 and 364 for the first three.
// Tried and no faster: two tiles in LDS and one barrier, no selects inside the last rows and channels, the first rows' loads before the
// weight's; loads and stores past the caches are slower (1 M rows 190 -> 213).
// The forward pass with a kink: 19 us, 55 and 109 for the same, where tiles take 22, 76 and 136; of few rows more (64 of 128 -> 128 5.2 against 3.7).
#include "layers.h"
#include "column_sum.h"

namespace cummhip {
namespace {

constexpr int kWaves = 8, kRows = kWaves * 16;

// element e of row r of a tile in LDS, P elements a row: 16-byte chunks apart as the transposing read wants them
template <int P>
__device__ __forceinline__ int turned(int r, int chunk) {
  constexpr int CPR = P / 8;
  const int swap = CPR >= 16 ? 2 * ((r & 3) + 4 * ((r >> 3) & 1)) : 2 * ((r & 3) ^ ((r >> 3) & 1));
  return (r * CPR + (chunk ^ swap)) * 16;
}
// lane's 8 rows, 8 q .. of those from `row` on, of column `col` (a multiple of 4, + what the other lanes of a group of 16 point to)
template <int P>
__device__ __forceinline__ v4i turning_read(const char *tile, int row, int col) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s *lds_v4s;
  const char *at = tile + turned<P>(row, col >> 3) + (col & 7) * 2, *next = tile + turned<P>(row + 4, col >> 3) + (col & 7) * 2;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)CUMM_LDS_PTR(at));
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)CUMM_LDS_PTR(next));
  return __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- which side of a kink an argument lies on.  Where the activation has one (at zero), its slope goes by the sign of z alone, and a
// gradient that passes or does not is no rounding: a z whose 32-bit sum lies within that sum's own error of zero is added up again
// in 64 bits (of 120 k rows, 64 -> 128 channels of ordinary numbers, one or two signs in ten such layers are wrong without).
// The error is at most (k + 8) 2^-23 of the sum of the products' magnitudes, in whatever order the matrix instructions add and
// whether they round or cut, and that sum at most the length of x's row times that of the weight's (Cauchy-Schwarz): one
// product and a comparison per element, and of ordinary numbers one element in 18000 (64 channels in) is that near.
// (bf16 rows whose squares leave 32 bits: above 1e19 all of a row is added up in 64, below 1e-19 it is left to its 32-bit sums.)
// the sum over the four lanes that share a row, lane & 15 alike (swaps of halves and quarters of a wave: no trip through LDS)
__device__ __forceinline__ uint2 four_swap(uint32_t v, bool halves) {
  const auto r = halves ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ float four_sum(float v) {
#pragma unroll
  for (int halves = 0; halves < 2; ++halves) {
    const uint2 r = four_swap(__builtin_bit_cast(uint32_t, v), halves);
    v = __builtin_bit_cast(float, r.x) + __builtin_bit_cast(float, r.y);
  }
  return v;
}
__device__ __forceinline__ double four_sum(double v) {
#pragma unroll
  for (int halves = 0; halves < 2; ++halves) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint2 lo = four_swap((uint32_t)b, halves), hi = four_swap((uint32_t)(b >> 32), halves);
    v = __builtin_bit_cast(double, (uint64_t)hi.x << 32 | lo.x) + __builtin_bit_cast(double, (uint64_t)hi.y << 32 | lo.y);
  }
  return v;
}

// The length of this lane's row (lane & 15) of a fragment's rows, of either operand: products of the rows with each other, of which a
// lane of the row's four has the row's own.  (The lengths' roundings are far below the 2^-6 that the bound has for them.)
template <class T, int KS, class Fragment>
__device__ __forceinline__ float row_length(Fragment fragment, int lane) {
  v4f own = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < KS; ++t) own = Elem<T>::mfma(fragment(t), fragment(t), own);
  const int i = lane & 15;
  const float sum = (i & 2) ? ((i & 1) ? own[3] : own[2]) : ((i & 1) ? own[1] : own[0]);
  return __builtin_amdgcn_sqrtf(four_sum((i >> 2) == (lane >> 4) ? sum : 0.0f));
}
// lengths[c] of the weight's rows, times what the bound is of them: a wave per block of 16
template <class T, int NP, int KP>
__device__ __forceinline__ void weight_lengths(const v4i (&w_z)[NP / 16][KP / 32][64], float (&lengths)[NP], int k, int wave, int lane) {
  for (int b = wave; b < NP / 16; b += kWaves) {
    const float length = row_length<T, KP / 32>([&](int t) { return w_z[b][t][lane]; }, lane);
    const int i = lane & 15;
    if (lane < 16) lengths[(b >> 1) * 32 + (i >> 2) * 8 + (b & 1) * 4 + (i & 3)] = length * ((float)(k + 8) * 0x1p-23f * 1.015625f);
  }
}

// z of 64 channels as the wave's lanes have it (this lane: row lane & 15, channels 8 (lane >> 4) .. of both runs of 32), made sure of.
// w_z, bias and lengths: of those channels.  The four lanes of a row add up one of its channels at a time, their own share of k each.
template <class T, int KS>
__device__ __forceinline__ void settle(v4f (&z)[2][2], const Piece<T> (&x)[KS], const v4i (*w_z)[KS][64], const float *bias, const float *lengths,
                                       float row, int lane) {
  const int q = lane >> 4;
  const auto over = [&](int s, int h, int e, const v4f &length) { return __builtin_fmaf(-row, length[e], __builtin_fabsf(z[s][h][e])); };
  float least = 1.0f;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v4f length = *reinterpret_cast<const v4f *>(lengths + s * 32 + q * 8 + h * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) least = __builtin_fminf(least, over(s, h, e, length));
    }
  if (__builtin_expect(__ballot(least < 0.0f) == 0, 1)) return;
  uint32_t mine = 0;      // bit 8 s + 4 h + e
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v4f length = *reinterpret_cast<const v4f *>(lengths + s * 32 + q * 8 + h * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) mine |= over(s, h, e, length) < 0.0f ? 1u << (s * 8 + h * 4 + e) : 0u;
    }
#pragma unroll 1
  while (__ballot(mine != 0) != 0) {
    // the first of the row's four lanes that has one left, and which: bit + 16 * its q
    uint32_t next = mine != 0 ? (uint32_t)__builtin_ctz(mine) + 16u * q : 64u;
#pragma unroll
    for (int halves = 0; halves < 2; ++halves) {
      const uint2 r = four_swap(next, halves);
      next = r.x < r.y ? r.x : r.y;
    }
    const bool own = next < 64u && (int)(next >> 4) == q;
    const int bit = next & 15, block = (bit >> 3) * 2 + (bit >> 2 & 1), place = (next >> 4 & 3) * 4 + (bit & 3);
    if (own) mine &= mine - 1;
    double sum = 0.0;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const v4i w = w_z[block][t][q * 16 + place];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t a = (uint32_t)w[d], b = (uint32_t)x[t].raw[d];
        asm volatile("" : "+v"(a), "+v"(b), "+v"(sum));      // (a pair of products after the other: together they need twice the registers)
        const float a0 = Elem<T>::to_float((uint16_t)a), b0 = Elem<T>::to_float((uint16_t)b);
        const float a1 = Elem<T>::to_float((uint16_t)(a >> 16)), b1 = Elem<T>::to_float((uint16_t)(b >> 16));
        if constexpr (std::is_same_v<T, F16>) {      // (products of those are exact in 32 bits)
          sum += (double)(a0 * b0);
          sum += (double)(a1 * b1);
        } else {
          sum = __builtin_fma((double)a0, (double)b0, sum);
          sum = __builtin_fma((double)a1, (double)b1, sum);
        }
      }
    }
    const float sure = (float)(four_sum(sum) + (double)bias[(bit >> 3) * 32 + (next >> 4 & 3) * 8 + (bit & 7)]);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[s][h][e] = own && bit == s * 8 + h * 4 + e ? sure : z[s][h][e];
  }
}

template <int NP> using GateBits = std::conditional_t<NP == 64, uint16_t, uint32_t>;

// The forward pass where the activation has a kink (with another one it is that of linear.h): the weight's fragments lie in LDS, a wave takes
// 16 rows through them, the next ones on their way.  What it decides it can leave as bits, for the backward pass: of a row, four numbers
// of NP / 4 bits, bit 8 s + e of the q-th for channel 32 s + 8 q + e, as the lanes have them.
template <class T, int NP, int KP, bool RESIDUAL>
__global__ __launch_bounds__(kWaves * 64, 4) void linear_narrow_forward_kernel(const LinearNarrowForward p, int waves) {
  using E = Elem<T>;
  constexpr int NS = NP / 32, KS = KP / 32;
  __shared__ v4i w_z[NP / 16][KS][64];
  __shared__ __attribute__((aligned(16))) float bias[NP], lengths[NP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  // (every lane loads on every path, as in the backward pass: behind the last row the last one, behind the last channel the first)
  Piece<T> x_next[KS];
  auto fetch = [&](int64_t first) __attribute__((always_inline)) {
    int64_t r = first + wave * 16 + l16;
    r = r < p.rows ? r : p.rows - 1;
#pragma unroll
    for (int s = 0; s < KS; ++s) x_next[s].load(p.x, r * p.ldx + (s * 32 + q * 8 < p.k ? s * 32 + q * 8 : 0), 8);
  };
  const bool relu = p.act == kActRelu;
  const int64_t stride = (int64_t)gridDim.x * waves * 16;
  int64_t first = (int64_t)blockIdx.x * waves * 16;
  fetch(first);
  constexpr int PER = (NP / 16) * KS / kWaves;
  Piece<T> v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int f = wave + j * kWaves, b = f / KS, s = f % KS, r = (b >> 1) * 32 + (l16 >> 2) * 8 + (b & 1) * 4 + (l16 & 3), c = s * 32 + q * 8;
    v[j].raw = v4i{0, 0, 0, 0};
    if (r < p.n && c < p.k) v[j].load(p.weight, (int64_t)r * p.ldw + c, 8);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int f = wave + j * kWaves, b = f / KS, s = f % KS;
    w_z[b][s][lane] = v[j].raw;
  }
  for (int c = threadIdx.x; c < NP; c += kWaves * 64) bias[c] = p.bias != nullptr && c < p.n ? E::to_float(reinterpret_cast<const uint16_t *>(p.bias)[c]) : 0.0f;
  __syncthreads();
  weight_lengths<T, NP, KP>(w_z, lengths, p.k, wave, lane);
  __syncthreads();
  if (wave >= waves) return;

  for (; first < p.rows; first += stride) {
    const int64_t r = first + wave * 16 + l16;
    const bool live = r < p.rows;
    Piece<T> x[KS], add_next[2];
    const auto fetch_add = [&](int s) __attribute__((always_inline)) {
      if constexpr (RESIDUAL) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = (s + u) * 32 + q * 8;
          add_next[u].load(p.residual, (live ? r : p.rows - 1) * p.ldr + (c < p.n ? c : 0), 8);
        }
      }
    };
    fetch_add(0);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s].raw[e] = live && s * 32 + q * 8 < p.k ? x_next[s].raw[e] : 0;
    fetch(first + stride);
    const float row = row_length<T, KS>([&](int t) { return x[t].raw; }, lane);
    uint32_t gate = 0;
#pragma unroll 1
    for (int s = 0; s < NS; s += 2) {      // a line of 128 bytes of a row
      const Piece<T> add[2] = {add_next[0], add_next[1]};
      fetch_add(s + 2 < NS ? s + 2 : 0);
      v4f z[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          z[u][h] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int t = 0; t < KS; ++t) z[u][h] = E::mfma(w_z[2 * (s + u) + h][t][lane], x[t].raw, z[u][h]);
          z[u][h] += *reinterpret_cast<const v4f *>(&bias[(s + u) * 32 + q * 8 + h * 4]);
        }
      settle<T, KS>(z, x, &w_z[2 * s], bias + s * 32, lengths + s * 32, row, lane);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = (s + u) * 32 + q * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[u][e >> 2][e & 3];
        const bool there = live && c < p.n;
        Piece<T> out;
#pragma unroll
        for (int e = 0; e < 8; ++e) gate |= v[e] <= 0.0f ? 0u : 1u << ((s + u) * 8 + e);      // (a NaN passes)
        if (p.pre != nullptr) {
          out.round(v);
          if (there) out.store(p.pre, r * p.ldp + c, 8);
        }
        if (p.out == nullptr) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.0f ? (relu ? 0.0f : v[e] * p.slope) : v[e];
        if constexpr (RESIDUAL) {
          float f[8];
          add[u].values(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += f[e];
        }
        out.round(v);
        if (there) out.store(p.out, r * p.ldo + c, 8);
      }
    }
    if (p.gate != nullptr && live) reinterpret_cast<GateBits<NP> *>(p.gate)[r * 4 + q] = (GateBits<NP>)gate;
  }
}

// The workgroup's LDS accesses before it are done, loads from memory stay on their way
__device__ __forceinline__ void wait_lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
  lds_barrier();
}

// GATE: the forward pass has left what passes as bits, z is not needed
template <class T, int NP, int KP, bool GATE>
__global__ __launch_bounds__(kWaves * 64) void linear_narrow_backward_kernel(const LinearNarrowParams p) {
  using E = Elem<T>;
  constexpr int NS = NP / 32, KS = KP / 32;
  __shared__ v4i w_z[GATE ? 1 : NP / 16][KS][64], w_x[KP / 16][NS][64], tile_z[kRows * NP / 8], tile_x[kRows * KP / 8];
  __shared__ __attribute__((aligned(16))) float bias[GATE ? 4 : NP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  const uint16_t *weight = reinterpret_cast<const uint16_t *>(p.weight);

  // the weight: as it lies (in the place of the rows' tile of dz), and from there both kinds of fragments
  char *raw = reinterpret_cast<char *>(tile_z);
  static_assert(KP <= kRows, "the weight fits there");
  for (int i = threadIdx.x; i < NP * KP / 8; i += kWaves * 64) {
    const int r = i / (KP / 8), c = i % (KP / 8);
    Piece<T> v;
    v.raw = v4i{0, 0, 0, 0};
    if (weight != nullptr && r < p.n && c * 8 < p.k) v.load(weight, (int64_t)r * p.ldw + c * 8, 8);
    *reinterpret_cast<v4i *>(raw + turned<KP>(r, c)) = v.raw;
  }
  for (int c = threadIdx.x; !GATE && c < NP; c += kWaves * 64) bias[c] = p.bias != nullptr && c < p.n ? E::to_float(reinterpret_cast<const uint16_t *>(p.bias)[c]) : 0.0f;
  __syncthreads();
  for (int f = wave; !GATE && f < (NP / 16) * KS; f += kWaves) {
    const int b = f / KS, s = f % KS, r = (b >> 1) * 32 + (l16 >> 2) * 8 + (b & 1) * 4 + (l16 & 3);
    w_z[b][s][lane] = *reinterpret_cast<const v4i *>(raw + turned<KP>(r, s * 4 + q));
  }
  for (int f = wave; f < (KP / 16) * NS; f += kWaves) {
    const int b = f / NS, s = f % NS;
    w_x[b][s][lane] = turning_read<KP>(raw, s * 32 + q * 8 + (l16 >> 2), (b >> 1) * 32 + (l16 & 3) * 8 + (b & 1) * 4);
  }
  __syncthreads();

  // blocks of grad_W: a block of 16 output channels a wave, or two waves to a block with half the input channels each
  constexpr int SPLIT = kWaves / (NP / 16), NB = KP / 16 / SPLIT;
  static_assert(SPLIT * NP == kWaves * 16 && SPLIT * NB * 16 == KP, "the waves share the blocks evenly");
  const int n_block = wave / SPLIT, k_block = (wave % SPLIT) * NB;
  v4f dw[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dw[b] = v4f{0, 0, 0, 0};
  float db[NS][8];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) db[s][e] = 0.0f;

  // Every lane loads on every path, so that the compiler can count them and waits for the rows before alone: behind the last row
  // the last one, behind the last channel the first ones (all of that becomes zeros below), instead of an x that is not there grad
  const void *const xs = p.x != nullptr ? p.x : p.grad;
  const int64_t ldx = p.x != nullptr ? p.ldx : p.ldg;
  const int k = p.x != nullptr ? p.k : 8;
  Piece<T> x_next[KS], g_next[NS];
  uint32_t gate_next = 0;
  auto fetch = [&](int64_t first) __attribute__((always_inline)) {
    int64_t r = first + wave * 16 + l16;
    r = r < p.rows ? r : p.rows - 1;
    if constexpr (GATE) gate_next = reinterpret_cast<const GateBits<NP> *>(p.gate)[r * 4 + q];
#pragma unroll
    for (int s = 0; s < KS; ++s) x_next[s].load(xs, r * ldx + (s * 32 + q * 8 < k ? s * 32 + q * 8 : 0), 8);
#pragma unroll
    for (int s = 0; s < NS; ++s) g_next[s].load(p.grad, r * p.ldg + (s * 32 + q * 8 < p.n ? s * 32 + q * 8 : 0), 8);
  };
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t first = (int64_t)blockIdx.x * kRows;
  fetch(first);
  for (; first < p.rows; first += stride) {
    Piece<T> x[KS], dz[NS];
#pragma unroll
    for (int s = 0; s < KS; ++s) x[s] = x_next[s];
#pragma unroll
    for (int s = 0; s < NS; ++s) dz[s] = g_next[s];
    [[maybe_unused]] const uint32_t gate = gate_next;
    fetch(first + stride);
    const int64_t r = first + wave * 16 + l16;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s].raw[e] = r < p.rows && s * 32 + q * 8 < p.k ? x[s].raw[e] : 0;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const bool there = r < p.rows && s * 32 + q * 8 < p.n;
      float g[8];
      dz[s].values(g);
      if constexpr (GATE) {
        const auto passes = [&](int e) { return (gate >> (s * 8 + e) & 1u) != 0; };
        if (p.act == kActRelu) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = passes(e) ? g[e] : 0.0f;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = passes(e) ? g[e] : g[e] * p.slope;
        }
      } else if (p.act != kActNone) {
        v4f z[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          z[h] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int t = 0; t < KS; ++t) z[h] = E::mfma(w_z[2 * s + h][t][lane], x[t].raw, z[h]);
          z[h] += *reinterpret_cast<const v4f *>(&bias[s * 32 + q * 8 + h * 4]);
        }
        linear_act_slopes(g, z[0], z[1], p.act, p.slope);
      }
      // (behind the last row and channel, an infinite or NaN operand's z is none: nothing of it may reach a product)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = there ? g[e] : 0.0f;
        db[s][e] += g[e];
      }
      dz[s].round(g);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (p.grad_x == nullptr) break;
      float f[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v4f acc = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NS; ++t) acc = E::mfma(w_x[2 * s + h][t][lane], dz[t].raw, acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[h * 4 + e] = acc[e];
      }
      Piece<T> out;
      out.round(f);
      if (r < p.rows && s * 32 + q * 8 < p.k) out.store(p.grad_x, r * p.k + s * 32 + q * 8, 8);
    }
    if (p.grad_weight == nullptr) continue;
    wait_lds_barrier();      // everybody has read the rows before these
#pragma unroll
    for (int s = 0; s < NS; ++s) *reinterpret_cast<v4i *>(reinterpret_cast<char *>(tile_z) + turned<NP>(wave * 16 + l16, s * 4 + q)) = dz[s].raw;
#pragma unroll
    for (int s = 0; s < KS; ++s) *reinterpret_cast<v4i *>(reinterpret_cast<char *>(tile_x) + turned<KP>(wave * 16 + l16, s * 4 + q)) = x[s].raw;
    wait_lds_barrier();
#pragma unroll
    for (int m = 0; m < kRows / 32; ++m) {
      const int row = m * 32 + q * 8 + (l16 >> 2), col = 4 * (l16 & 3);
      const v4i z = turning_read<NP>(reinterpret_cast<const char *>(tile_z), row, n_block * 16 + col);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        dw[b] = E::mfma(turning_read<KP>(reinterpret_cast<const char *>(tile_x), row, (k_block + b) * 16 + col), z, dw[b]);
    }
  }

  // this workgroup's sums: grad_W [NP][KP], grad_b [NP] (over the 16 rows of a wave's lanes, then over the waves in order)
  float *to = p.partial + (int64_t)blockIdx.x * (NP * KP + NP);
  if (p.grad_weight != nullptr) {
#pragma unroll
    for (int b = 0; b < NB; ++b) *reinterpret_cast<v4f *>(to + (n_block * 16 + l16) * KP + (k_block + b) * 16 + q * 4) = dw[b];
  }
  if (p.grad_bias == nullptr) return;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int d = 1; d < 16; d *= 2) db[s][e] += __shfl_xor(db[s][e], d);
  __syncthreads();      // the last rows' tiles have been read
  float(*waves)[NP] = reinterpret_cast<float(*)[NP]>(tile_z);
  if (l16 == 0) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) waves[wave][s * 32 + q * 8 + e] = db[s][e];
  }
  __syncthreads();
  if (threadIdx.x < NP) {
    float sum = waves[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += waves[w][threadIdx.x];
    to[NP * KP + threadIdx.x] = sum;
  }
}

// the workgroups' sums, 16 columns a workgroup: those of grad_W, then those of grad_b
template <class T>
__global__ __launch_bounds__(256) void linear_narrow_sum_kernel(const LinearNarrowParams p, int blocks, int np, int kp) {
  const int c0 = blockIdx.x * 16, c = c0 + (int)threadIdx.x;
  const bool of_bias = c0 >= np * kp;
  if (of_bias ? c0 - np * kp >= p.n : p.grad_weight == nullptr || c0 / kp >= p.n || c0 % kp >= p.k) return;
  const float total = column_final_sum(p.partial, np * kp + np, 0, blocks, blockIdx.x);
  if (threadIdx.x >= 16) return;
  const uint16_t v = Elem<T>::from_float(total);
  if (of_bias) {
    if (c - np * kp < p.n) reinterpret_cast<uint16_t *>(p.grad_bias)[c - np * kp] = v;
  } else if (c % kp < p.k) {
    reinterpret_cast<uint16_t *>(p.grad_weight)[(c / kp) * p.k + c % kp] = v;
  }
}

// a workgroup per CU (its LDS), rows for each at least
int narrow_blocks(int64_t rows) {
  const int64_t groups = (rows + kRows - 1) / kRows;
  return (int)(groups < 256 ? groups : 256);
}
int padded(int channels) { return channels <= 64 ? 64 : 128; }

template <class T>
hipError_t launch(const LinearNarrowParams &p, int blocks, hipStream_t s) {
  const int np = padded(p.n), kp = padded(p.k);
  const auto run = [&](auto plain, auto gated) { hipLaunchKernelGGL(p.gate != nullptr ? gated : plain, dim3((unsigned)blocks), dim3(kWaves * 64), 0, s, p); };
#define CUMM_NARROW(NP, KP) run(linear_narrow_backward_kernel<T, NP, KP, false>, linear_narrow_backward_kernel<T, NP, KP, true>)
  if (np == 64) kp == 64 ? CUMM_NARROW(64, 64) : CUMM_NARROW(64, 128);
  else kp == 64 ? CUMM_NARROW(128, 64) : CUMM_NARROW(128, 128);
#undef CUMM_NARROW
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (p.grad_weight == nullptr && p.grad_bias == nullptr)) return e;
  hipLaunchKernelGGL(linear_narrow_sum_kernel<T>, dim3((unsigned)((np * kp + (p.grad_bias ? np : 0)) / 16)), dim3(256), 0, s, p, blocks, np, kp);
  return hipGetLastError();
}

template <class T>
hipError_t launch(const LinearNarrowForward &p, hipStream_t s) {
  const int np = padded(p.n), kp = padded(p.k);
  // Few rows: so many waves of a workgroup have some as it takes to use the CUs, all of them fetch the weight (1000 rows, 64 -> 128: 5.6 us, with eight of them 6.1).
  // Two workgroups per CU, which is what its registers allow
  int waves = 1;
  while (waves < kWaves && (p.rows + waves * 16 - 1) / (waves * 16) > 256) waves *= 2;
  const int64_t groups = (p.rows + waves * 16 - 1) / (waves * 16);
  const unsigned blocks = (unsigned)(groups < 512 ? groups : 512);
  const auto run = [&](auto with, auto without) { hipLaunchKernelGGL(p.residual != nullptr ? with : without, dim3(blocks), dim3(kWaves * 64), 0, s, p, waves); };
#define CUMM_NARROW(NP, KP) run(linear_narrow_forward_kernel<T, NP, KP, true>, linear_narrow_forward_kernel<T, NP, KP, false>)
  if (np == 64) kp == 64 ? CUMM_NARROW(64, 64) : CUMM_NARROW(64, 128);
  else kp == 64 ? CUMM_NARROW(128, 64) : CUMM_NARROW(128, 128);
#undef CUMM_NARROW
  return hipGetLastError();
}

}  // namespace

bool linear_narrow_forward_takes(int n, int k, int act) {
  return n % 8 == 0 && k % 8 == 0 && n <= kLinearNarrow && k <= kLinearNarrow && (act == kActRelu || act == kActLeakyRelu);
}
hipError_t launch_linear_narrow_forward(const LinearNarrowForward &p, bool bf16, hipStream_t s) { return bf16 ? launch<BF16>(p, s) : launch<F16>(p, s); }

int64_t linear_narrow_gate_bytes(int64_t rows, int n) { return rows * (padded(n) / 8); }
int64_t linear_narrow_bytes(int64_t rows, int n, int k) { return (int64_t)narrow_blocks(rows) * padded(n) * (padded(k) + 1) * 4; }
hipError_t launch_linear_narrow_backward(const LinearNarrowParams &p, bool bf16, hipStream_t s) {
  return bf16 ? launch<BF16>(p, narrow_blocks(p.rows), s) : launch<F16>(p, narrow_blocks(p.rows), s);
}

}  // namespace cummhip
