// Host side of the row-wise layers: products with an epilogue (linear_inst.hip) and norms (rownorm_inst.hip)
#pragma once
#include "linear.h"

namespace cummhip {

// the calling thread's last error (cumm_hip_last_error); returns code
int layer_error(int code, const char *what);

// ---- products
enum LinearLayout { kResult = 0, kGradInput = 1, kGradWeight = 2 };      // (XT, YT) = (0, 0), (1, 0), (1, 1)
// Which kernel, and into how many slices the contraction is cut
struct LinearPlan {
  int tile;      // kTile*
  int slices;
  double us;     // its estimated time
};
enum LinearTile { kTileFew = 0, kTile64 = 1, kTile64x128 = 2, kTile128 = 3, kTile128x256 = 4, kTile256 = 5, kTile64Small = 6, kTileAny = 7 };
// k in units of two bytes
LinearPlan linear_plan(LinearLayout layout, int64_t m, int n, int64_t k);
LinearPlan linear_plan_any(const LinearPlan &plan, int64_t m, int n, int64_t k, int64_t copied);
// whether its launch stays below 2^32 threads
bool linear_plan_fits(const LinearPlan &plan, int64_t m, int n);
// bytes of the slices' sums (0 = one slice)
inline int64_t linear_partial_bytes(const LinearPlan &plan, int64_t m, int n) {
  return plan.slices > 1 ? (int64_t)plan.slices * m * ((n + 7) / 8 * 8) * 4 : 0;
}
hipError_t launch_linear_f16(LinearLayout layout, const LinearPlan &plan, const LinearParams &p, hipStream_t s);
hipError_t launch_linear_bf16(LinearLayout layout, const LinearPlan &plan, const LinearParams &p, hipStream_t s);
// 8-bit operands, output f16 or bf16 (layout kResult)
hipError_t launch_linear_s8(bool bf16, const LinearPlan &plan, const LinearParams &p, hipStream_t s);
hipError_t launch_linear_repack(LinearRepack p, int elem_bytes, hipStream_t s);      // (pieces and wgs are filled in)

struct LinearGateParams {
  const void *grad;        // [rows, n]
  const void *pre;         // [rows, n] what the activation got, NULL = it is none
  void *dz;                // [rows, ldz], NULL = sums only
  int64_t ldg, ldp, ldz;   // elements; ldz: those of a row that are written, n rounded up to 8
  int64_t dz_pitch;
  float *partial;          // [blocks, pitch], NULL = no sums
  int64_t rows, rows_per_block;
  int32_t n, pitch, shift, act;
  float slope;
};
void linear_gate_shape(int64_t rows, int n, int *shift, int *strips, int *blocks, int64_t *per);
hipError_t launch_linear_gate(LinearGateParams p, int64_t dz_pitch, void *grad_bias, bool bf16, hipStream_t s);
// The whole backward pass of n and k up to kLinearNarrow, multiples of 8 (linear_narrow_inst.hip)
constexpr int kLinearNarrow = 128;
struct LinearNarrowParams {
  const void *x, *grad, *weight, *bias;      // [rows, k], [rows, n], [n, k], [n] or NULL; x and weight NULL where nothing wants them
  void *grad_x, *grad_weight, *grad_bias;    // dense; each may be NULL
  float *partial;                            // linear_narrow_bytes
  const void *gate;                          // of an activation with a kink, as the forward pass leaves it; NULL of any other
  int64_t rows, ldx, ldg, ldw;               // elements
  int32_t n, k, act;
  float slope;
};
// The forward pass of the same layers where the activation has a kink
struct LinearNarrowForward {
  const void *x, *weight, *bias, *residual;      // [rows, k], [n, k], [n] or NULL, [rows, n] or NULL
  void *out, *pre, *gate;                        // [rows, n], [rows, n] and linear_narrow_gate_bytes; each may be NULL
  int64_t rows, ldx, ldw, ldr, ldo, ldp;         // elements
  int32_t n, k, act;
  float slope;
};
int64_t linear_narrow_gate_bytes(int64_t rows, int n);
bool linear_narrow_forward_takes(int n, int k, int act);
hipError_t launch_linear_narrow_forward(const LinearNarrowForward &p, bool bf16, hipStream_t s);
int64_t linear_narrow_bytes(int64_t rows, int n, int k);
hipError_t launch_linear_narrow_backward(const LinearNarrowParams &p, bool bf16, hipStream_t s);
// two-byte elements (a kernel: memset nodes of captured graphs have given wrong results on replays)
hipError_t launch_rows_zero(void *dst, int64_t elements, hipStream_t s);

// ---- norms
struct NormParams {
  const void *x, *residual;      // rows of k elements; residual may be NULL
  const void *weight;            // [k]; NULL = no norm
  void *out, *total;             // [rows, k]
  int8_t *codes;                 // [rows, k] instead of out
  float *scale, *inv;            // [rows]; inv may be NULL
  int64_t rows, ldx, ldr;
  int32_t k;
  float eps;
};
hipError_t launch_norm(const NormParams &p, int dtype, hipStream_t s);
struct NormGradParams {
  const void *h, *weight, *grad, *grad_total;      // grad or grad_total may be NULL: zeros
  const float *inv;
  void *grad_in;           // [rows, k], may be NULL
  void *grad_weight;       // [k]
  float *partial;          // [blocks, pitch]; NULL = no grad_weight
  int64_t rows, ldh, ldg, ldt;
  int32_t k, pitch, blocks;
};
int norm_backward_blocks(int64_t rows, int k);
hipError_t launch_norm_backward(const NormGradParams &p, bool bf16, hipStream_t s);

}  // namespace cummhip
