// The backward pass of a layer with few channels on both sides, in one pass over its rows:
//     z = x W^T + b (f32, worked out again: the forward pass writes nothing for it),  dz = grad act'(z) (rounded for the products),
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
// Measured with ReLU and all gradients, both launches, against the gate and two products (which read a stored z): 119985 rows, 64 ->
// 128 channels, f16, 29.9 us against 50.8 (and the forward pass 22 against 26 without z to write); 1 M rows, 64 -> 64 78 against 171 (4.9 TB/s
// of what it moves), 128 -> 128 190 against 364 (4.0); 1000 rows 13 against 20.  With gelu 1 M rows, 128 -> 128 take 230: 25 instructions an element,
// which the loads do not hide.  Tried and no faster: two tiles in LDS and one barrier (30.1), no selects inside the last rows and
// channels (30.1), the first rows' loads before the weight's (30.2); loads and stores past the caches are slower (1 M rows 190 -> 213).
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

// The workgroup's LDS accesses before it are done, loads from memory stay on their way
__device__ __forceinline__ void wait_lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
  lds_barrier();
}

template <class T, int NP, int KP>
__global__ __launch_bounds__(kWaves * 64) void linear_narrow_backward_kernel(const LinearNarrowParams p) {
  using E = Elem<T>;
  constexpr int NS = NP / 32, KS = KP / 32;
  __shared__ v4i w_z[NP / 16][KS][64], w_x[KP / 16][NS][64], tile_z[kRows * NP / 8], tile_x[kRows * KP / 8];
  __shared__ __attribute__((aligned(16))) float bias[NP];
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
  for (int c = threadIdx.x; c < NP; c += kWaves * 64) bias[c] = p.bias != nullptr && c < p.n ? E::to_float(reinterpret_cast<const uint16_t *>(p.bias)[c]) : 0.0f;
  __syncthreads();
  for (int f = wave; f < (NP / 16) * KS; f += kWaves) {
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
  auto fetch = [&](int64_t first) __attribute__((always_inline)) {
    int64_t r = first + wave * 16 + l16;
    r = r < p.rows ? r : p.rows - 1;
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
      if (p.act != kActNone) {
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
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kWaves * 64), 0, s, p); };
  if (np == 64) kp == 64 ? run(linear_narrow_backward_kernel<T, 64, 64>) : run(linear_narrow_backward_kernel<T, 64, 128>);
  else kp == 64 ? run(linear_narrow_backward_kernel<T, 128, 64>) : run(linear_narrow_backward_kernel<T, 128, 128>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (p.grad_weight == nullptr && p.grad_bias == nullptr)) return e;
  hipLaunchKernelGGL(linear_narrow_sum_kernel<T>, dim3((unsigned)((np * kp + (p.grad_bias ? np : 0)) / 16)), dim3(256), 0, s, p, blocks, np, kp);
  return hipGetLastError();
}

}  // namespace

int64_t linear_narrow_bytes(int64_t rows, int n, int k) { return (int64_t)narrow_blocks(rows) * padded(n) * (padded(k) + 1) * 4; }
hipError_t launch_linear_narrow_backward(const LinearNarrowParams &p, bool bf16, hipStream_t s) {
  return bf16 ? launch<BF16>(p, narrow_blocks(p.rows), s) : launch<F16>(p, narrow_blocks(p.rows), s);
}

}  // namespace cummhip
