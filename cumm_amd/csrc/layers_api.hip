// C entry points of the row-wise layers: argument checks, the layout of the workspace, launches.
#include "../../include/cumm_hip.h"

#include "layers.h"

using namespace cummhip;

namespace {

int bad(const char *what) { return layer_error(CUMM_HIP_EINVAL, what); }
int launched(hipError_t e) { return e == hipSuccess ? CUMM_HIP_OK : layer_error(CUMM_HIP_ERUNTIME, hipGetErrorString(e)); }

bool two_byte(int dt) { return dt == CUMM_HIP_F16 || dt == CUMM_HIP_BF16; }
bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool on(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

constexpr int64_t kRowBytes = (int64_t)8 << 20;      // 256 rows of a tile lie within 2^31 bytes
constexpr int64_t kMaxRows = 0x7fffffff;
constexpr int kMaxWhole = 131071;                    // 8-bit operands: k * 128 * 128 < 2^31

// Pieces of the workspace in the order they are asked for: their sum, and, once there is a base, their places
struct Workspace {
  char *base;
  int64_t used = 0;
  void *take(int64_t bytes) {
    void *at = base ? base + used : nullptr;
    used += up(bytes, 256);
    return at;
  }
};

// A matrix operand as the products read it: its own rows where they lie on 16-byte borders and are whole 16-byte pieces long,
// else a copy of them (lines of 128 bytes apart) in the workspace
struct Operand {
  const void *from;
  int64_t rows, cols, ld;      // elements
  int bytes;                   // of one
  void *copy = nullptr;
  bool direct() const { return on16(from) && ld * bytes % 16 == 0 && cols * bytes % 16 == 0; }
  int64_t pitch() const { return direct() ? ld * bytes : up(cols * bytes, 128); }
  const void *at() const { return direct() ? from : copy; }
  void place(Workspace &w) {
    if (!direct()) copy = w.take(rows * pitch());
  }
  LinearRepack::One repack() const { return direct() ? LinearRepack::One{} : LinearRepack::One{copy, from, rows, cols, ld, pitch(), 0, 0}; }
};
hipError_t fill(const Operand &a, const Operand &b, hipStream_t s) {
  return a.direct() && b.direct() ? hipSuccess : launch_linear_repack(LinearRepack{{a.repack(), b.repack()}}, a.bytes, s);
}

// Layers of few channels whose activation has a kink: rows and weight at any address, no workspace, and a gate for the backward pass
bool narrow_forward(const CummHipLinearArgs &a) { return a.dtype != CUMM_HIP_S8 && linear_narrow_forward_takes(a.n, a.k, a.act_type); }
bool narrow_gate(const CummHipLinearGradArgs &a) { return a.from_inputs && linear_narrow_forward_takes(a.n, a.k, a.act_type); }

constexpr int kMaxRow = 1 << 30;                     // elements of a row of a norm

const char *linear_checked(const CummHipLinearArgs &a) {
  const bool s8 = a.dtype == CUMM_HIP_S8;
  if (!s8 && !two_byte(a.dtype)) return "linear: operands are f16, bf16 or s8";
  if (s8 ? !two_byte(a.out_dtype) : a.out_dtype != a.dtype) return "linear: the output is f16 or bf16, that of the operands unless they are s8";
  if (a.m < 0 || a.m > kMaxRows || a.n < 1 || a.k < 1) return "linear: m, n and k must not be empty (m may be 0) or exceed int32 range";
  const int size = s8 ? 1 : 2;
  if (a.ld_x < a.k || a.ld_weight < a.k || a.ld_out < a.n || (a.residual && a.ld_residual < a.n) || (a.pre_act && a.ld_pre_act < a.n))
    return "linear: rows overlap (a pitch is smaller than its row)";
  if (a.ld_x * size >= kRowBytes || a.ld_weight * size >= kRowBytes || up((int64_t)a.k * size, 128) >= kRowBytes) return "linear: rows of 8 MiB and more are not taken";
  if (s8 && a.k > kMaxWhole) return "linear: sums of more than 131071 products of 8 bits may exceed int32 range";
  if (a.act_type < 0 || a.act_type > CUMM_HIP_ACT_GELU_TANH) return "linear: unknown activation";
  if (a.gate && !narrow_forward(a)) return "linear: a gate is left by two-byte layers of few channels with a ReLU or leaky ReLU";
  if (a.m == 0) return nullptr;
  if (!a.x || !a.weight || !a.out) return "linear: x, weight and out must not be null";
  if (s8 && (!a.x_scale || !a.weight_scale)) return "linear: 8-bit operands need the scales of their rows";
  if (!on(a.x, size) || !on(a.weight, size) || !on(a.out, 2) || !on(a.residual, 2) || !on(a.pre_act, 2) || !on(a.bias, s8 ? 4 : 2) || !on(a.gate, 4) ||
      (s8 && (!on(a.x_scale, 4) || !on(a.weight_scale, 4))))
    return "linear: a pointer is not aligned to its elements";
  return nullptr;
}

struct LinearCall {
  Operand x, weight;
  LinearPlan plan;
  int64_t k2;      // k in units of two bytes, as the copies have it
  bool fits, any;  // any: the operands as they lie, whatever their alignment
  void *partial;
  LinearCall(const CummHipLinearArgs &a, Workspace &w) {
    const int size = a.dtype == CUMM_HIP_S8 ? 1 : 2;
    x = {a.x, a.m, a.k, a.ld_x, size};
    weight = {a.weight, a.n, a.k, a.ld_weight, size};
    k2 = up((int64_t)a.k * size, 16) / 2;
    plan = linear_plan(kResult, a.m, a.n, k2);
    if ((!x.direct() || !weight.direct()) && (int64_t)a.k * size >= 16) {      // (a piece lies inside its row)
      plan = linear_plan_any(plan, a.m, a.n, k2, ((x.direct() ? 0 : x.rows) + (weight.direct() ? 0 : weight.rows)) * a.k * size);
    }
    any = plan.tile == kTileAny;
    if (!any) {
      x.place(w);
      weight.place(w);
    }
    fits = linear_plan_fits(plan, a.m, a.n);
    partial = plan.slices > 1 ? w.take(linear_partial_bytes(plan, a.m, a.n)) : nullptr;
  }
};
constexpr char kTooMany[] = "linear: too many outputs for one launch";

hipError_t launch_two_byte(int dtype, LinearLayout layout, const LinearPlan &plan, const LinearParams &p, hipStream_t s) {
  return dtype == CUMM_HIP_BF16 ? launch_linear_bf16(layout, plan, p, s) : launch_linear_f16(layout, plan, p, s);
}

const char *linear_grad_checked(const CummHipLinearGradArgs &a) {
  if (!two_byte(a.dtype)) return "linear backward: f16 or bf16";
  if (a.m < 0 || a.m > kMaxRows || a.n < 1 || a.k < 1) return "linear backward: m, n and k must not be empty (m may be 0) or exceed int32 range";
  if (a.act_type < 0 || a.act_type > CUMM_HIP_ACT_GELU_TANH) return "linear backward: unknown activation";
  if (a.ld_grad_out < a.n || (a.pre_act && a.ld_pre_act < a.n) || (a.x && a.ld_x < a.k) || (a.weight && a.ld_weight < a.k))
    return "linear backward: rows overlap (a pitch is smaller than its row)";
  const int64_t most = kRowBytes / 2;
  if (a.ld_grad_out >= most || a.ld_x >= most || a.ld_weight >= most || up(a.n, 64) >= most || up(a.k, 64) >= most)
    return "linear backward: rows of 8 MiB and more are not taken";
  if (a.m == 0) return nullptr;
  if (a.grad_x && !a.weight) return "linear backward: the gradient of x needs the weight";
  if (a.grad_weight && !a.x) return "linear backward: the gradient of the weight needs x";
  if (!a.grad_out) return "linear backward: grad_out must not be null";
  if (a.from_inputs) {
    if (a.n % 8 || a.k % 8 || a.n > kLinearNarrow || a.k > kLinearNarrow) return "linear backward: from the inputs only where n and k are multiples of 8, up to 128";
    if (a.act_type != CUMM_HIP_ACT_NONE && !a.gate && (!a.x || !a.weight)) return "linear backward: from the inputs, x and weight must not be null";
    if (a.gate && !narrow_gate(a)) return "linear backward: a gate is that of a ReLU or leaky ReLU";
    if (!on(a.gate, 4)) return "linear backward: a pointer is not aligned to its elements";
  } else if (a.gate) {
    return "linear backward: a gate goes with from_inputs";
  } else if (a.act_type != CUMM_HIP_ACT_NONE && !a.pre_act) return "linear backward: the activation's argument (pre_act) is missing";
  for (const void *p : {a.grad_out, a.pre_act, a.x, a.weight, a.bias, (const void *)a.grad_x, (const void *)a.grad_weight, (const void *)a.grad_bias})
    if (!on(p, 2)) return "linear backward: a pointer is not aligned to its elements";
  return nullptr;
}

struct LinearGradCall {
  Operand x = {nullptr, 0, 0, 0, 2}, weight = x;      // (none, and so in place)
  LinearGateParams gate = {};
  bool gated;              // a launch that writes dz, or the bias sums, or both
  const void *dz;
  int64_t ldz;             // elements
  LinearPlan plan_x = {0, 1, 0}, plan_w = {0, 1, 0};
  void *partial_x = nullptr, *partial_w = nullptr;
  bool fits = true;
  LinearGradCall(const CummHipLinearGradArgs &a, Workspace &w) {
    const bool act = a.act_type != CUMM_HIP_ACT_NONE, products = a.grad_x || a.grad_weight;
    const Operand g = {a.grad_out, a.m, a.n, a.ld_grad_out, 2};
    const bool write = products && (act || !g.direct());
    gated = write || a.grad_bias;
    dz = a.grad_out;
    ldz = a.ld_grad_out;
    gate.grad = a.grad_out;
    gate.pre = act ? a.pre_act : nullptr;
    gate.ldg = a.ld_grad_out;
    gate.ldp = a.ld_pre_act;
    gate.rows = a.m;
    gate.n = a.n;
    gate.act = a.act_type;
    gate.slope = a.act_alpha;
    gate.pitch = (int)up(a.n, 16);
    if (write) {
      ldz = up(a.n, a.n >= 64 ? 64 : 8);
      dz = gate.dz = w.take(a.m * ldz * 2);
      gate.ldz = up(a.n, 8);      // (what is written of a row; its pitch is ldz)
    }
    if (a.grad_bias) {
      int shift, strips, blocks;
      int64_t per;
      linear_gate_shape(a.m, a.n, &shift, &strips, &blocks, &per);
      gate.partial = reinterpret_cast<float *>(w.take((int64_t)blocks * gate.pitch * 4));
    }
    if (a.grad_x) {
      weight = {a.weight, a.n, a.k, a.ld_weight, 2};
      weight.place(w);
      plan_x = linear_plan(kGradInput, a.m, a.k, a.n);
      fits = linear_plan_fits(plan_x, a.m, a.k);
      if (plan_x.slices > 1) partial_x = w.take(linear_partial_bytes(plan_x, a.m, a.k));
    }
    if (a.grad_weight) {
      x = {a.x, a.m, a.k, a.ld_x, 2};
      x.place(w);
      plan_w = linear_plan(kGradWeight, a.n, a.k, a.m);
      fits = fits && linear_plan_fits(plan_w, a.n, a.k);
      if (plan_w.slices > 1) partial_w = w.take(linear_partial_bytes(plan_w, a.n, a.k));
    }
  }
};

const char *norm_checked(const CummHipRmsNormArgs &a) {
  const bool norm = a.weight != nullptr;
  if (!two_byte(a.dtype) && !(a.dtype == CUMM_HIP_F32 && !norm && !a.out)) return "rms norm: f16 or bf16 (f32 for rows in 8 bits without a norm)";
  if (a.m < 0 || a.m > kMaxRows || a.k < 1) return "rms norm: rows must not be empty, their number must not exceed int32 range";
  if (a.k > kMaxRow) return "rms norm: rows of more than 2^30 elements are not taken";
  if (a.ld_x < a.k || (a.residual && a.ld_residual < a.k)) return "rms norm: rows overlap (a pitch is smaller than its row)";
  if (norm && !(a.eps > 0.0f)) return "rms norm: eps must be positive";
  if (!norm && (a.residual || a.total || a.inv_rms)) return "rms norm: no residual, sum or statistics without a norm";
  if ((a.residual != nullptr) != (a.total != nullptr) && a.m > 0) return "rms norm: the sum is written where there is a residual, and only there";
  if (a.m == 0) return nullptr;
  if (!a.x || (a.out != nullptr) == (a.codes != nullptr)) return "rms norm: x, and either out or codes, must not be null";
  if (!norm && !a.codes) return "rms norm: a norm needs its weight";
  if ((a.codes != nullptr) != (a.scale != nullptr)) return "rms norm: a scale per row goes with 8-bit rows";
  const int size = a.dtype == CUMM_HIP_F32 ? 4 : 2;
  if (!on(a.x, size) || !on(a.residual, 2) || !on(a.weight, 2) || !on(a.out, 2) || !on(a.total, 2) || !on(a.scale, 4) || !on(a.inv_rms, 4))
    return "rms norm: a pointer is not aligned to its elements";
  return nullptr;
}

const char *norm_grad_checked(const CummHipRmsNormGradArgs &a) {
  if (!two_byte(a.dtype)) return "rms norm backward: f16 or bf16";
  if (a.m < 0 || a.m > kMaxRows || a.k < 1) return "rms norm backward: rows must not be empty, their number must not exceed int32 range";
  if (a.k > kMaxRow) return "rms norm backward: rows of more than 2^30 elements are not taken";
  if (a.ld_total < a.k || (a.grad_out && a.ld_grad_out < a.k) || (a.grad_total && a.ld_grad_total < a.k))
    return "rms norm backward: rows overlap (a pitch is smaller than its row)";
  if (a.m == 0) return nullptr;
  if (!a.total || !a.weight || !a.inv_rms) return "rms norm backward: total, weight and inv_rms must not be null";
  for (const void *p : {a.total, a.weight, a.grad_out, a.grad_total, (const void *)a.grad_x, (const void *)a.grad_weight})
    if (!on(p, 2)) return "rms norm backward: a pointer is not aligned to its elements";
  if (!on(a.inv_rms, 4)) return "rms norm backward: a pointer is not aligned to its elements";
  return nullptr;
}

const char *workspace_checked(const void *workspace, size_t bytes, int64_t need) {
  if (need == 0) return nullptr;
  if (!workspace || (int64_t)bytes < need) return "the workspace is smaller than cumm_hip_*_workspace says";
  return on(workspace, 256) ? nullptr : "the workspace must be 256-byte aligned";
}

}  // namespace

extern "C" {

int64_t cumm_hip_linear_workspace(const CummHipLinearArgs *a) {
  if (!a || linear_checked(*a)) return -1;
  if (a->m == 0 || narrow_forward(*a)) return 0;
  Workspace w = {nullptr};
  const LinearCall call(*a, w);
  return call.fits ? w.used : -1;
}

int cumm_hip_linear(const CummHipLinearArgs *a, void *stream) {
  if (!a) return bad("linear: null arguments");
  if (const char *e = linear_checked(*a)) return bad(e);
  if (a->m == 0) return CUMM_HIP_OK;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (narrow_forward(*a)) {
    const LinearNarrowForward p = {a->x, a->weight, a->bias, a->residual, a->out, a->pre_act, a->gate, a->m, a->ld_x, a->ld_weight, a->ld_residual,
                                   a->ld_out, a->ld_pre_act, a->n, a->k, a->act_type, a->act_alpha};
    return launched(launch_linear_narrow_forward(p, a->dtype == CUMM_HIP_BF16, s));
  }
  Workspace w = {reinterpret_cast<char *>(a->workspace)};
  const LinearCall call(*a, w);
  if (!call.fits) return bad(kTooMany);
  if (const char *e = workspace_checked(a->workspace, a->workspace_bytes, w.used)) return bad(e);
  const hipError_t e = call.any ? hipSuccess : fill(call.x, call.weight, s);
  if (e != hipSuccess) return launched(e);
  LinearParams p = {};
  p.X = call.any ? a->weight : call.weight.at();
  p.Y = call.any ? a->x : call.x.at();
  p.ldx = call.any ? a->ld_weight * call.x.bytes : call.weight.pitch();
  p.ldy = call.any ? a->ld_x * call.x.bytes : call.x.pitch();
  p.row_bytes = a->k * call.x.bytes;
  p.m = a->m;
  p.n = a->n;
  p.k = call.k2;
  p.out = a->out;
  p.ldo = a->ld_out;
  p.bias = a->bias;
  p.residual = a->residual;
  p.ldr = a->ld_residual;
  p.pre = a->pre_act;
  p.ldp = a->ld_pre_act;
  p.y_scale = a->x_scale;
  p.x_scale = a->weight_scale;
  p.act = a->act_type;
  p.slope = a->act_alpha;
  p.partial = call.partial;
  p.slices = call.plan.slices;
  if (a->dtype == CUMM_HIP_S8) return launched(launch_linear_s8(a->out_dtype == CUMM_HIP_BF16, call.plan, p, s));
  return launched(launch_two_byte(a->dtype, kResult, call.plan, p, s));
}

int64_t cumm_hip_linear_backward_workspace(const CummHipLinearGradArgs *a) {
  if (!a || linear_grad_checked(*a)) return -1;
  if (a->m == 0) return 0;
  if (a->from_inputs) {
    return up(linear_narrow_bytes(a->m, a->n, a->k), 256) + (narrow_gate(*a) && !a->gate ? up(linear_narrow_gate_bytes(a->m, a->n), 256) : 0);
  }
  Workspace w = {nullptr};
  const LinearGradCall call(*a, w);
  return call.fits ? w.used : -1;
}

int cumm_hip_linear_backward(const CummHipLinearGradArgs *a, void *stream) {
  if (!a) return bad("linear backward: null arguments");
  if (const char *e = linear_grad_checked(*a)) return bad(e);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->m == 0) {
    hipError_t e = a->grad_weight ? launch_rows_zero(a->grad_weight, (int64_t)a->n * a->k, s) : hipSuccess;
    if (e == hipSuccess && a->grad_bias) e = launch_rows_zero(a->grad_bias, a->n, s);
    return launched(e);
  }
  if (a->from_inputs) {
    if (const char *e = workspace_checked(a->workspace, a->workspace_bytes, cumm_hip_linear_backward_workspace(a))) return bad(e);
    if (!a->grad_x && !a->grad_weight && !a->grad_bias) return CUMM_HIP_OK;
    const bool bf16 = a->dtype == CUMM_HIP_BF16;
    const void *gate = a->gate;
    if (narrow_gate(*a) && !gate) {      // nobody has kept it: a forward pass for it alone
      void *made = reinterpret_cast<char *>(a->workspace) + up(linear_narrow_bytes(a->m, a->n, a->k), 256);
      const LinearNarrowForward p = {a->x, a->weight, a->bias, nullptr, nullptr, nullptr, made, a->m, a->ld_x, a->ld_weight, 0, 0, 0, a->n, a->k, a->act_type, a->act_alpha};
      const hipError_t e = launch_linear_narrow_forward(p, bf16, s);
      if (e != hipSuccess) return launched(e);
      gate = made;
    }
    const LinearNarrowParams p = {a->x, a->grad_out, a->weight, a->bias, a->grad_x, a->grad_weight, a->grad_bias, reinterpret_cast<float *>(a->workspace),
                                  gate, a->m, a->ld_x, a->ld_grad_out, a->ld_weight, a->n, a->k, a->act_type, a->act_alpha};
    return launched(launch_linear_narrow_backward(p, bf16, s));
  }
  Workspace w = {reinterpret_cast<char *>(a->workspace)};
  const LinearGradCall call(*a, w);
  if (!call.fits) return bad(kTooMany);
  if (const char *e = workspace_checked(a->workspace, a->workspace_bytes, w.used)) return bad(e);
  const bool bf16 = a->dtype == CUMM_HIP_BF16;
  hipError_t e = call.gated ? launch_linear_gate(call.gate, call.ldz, a->grad_bias, bf16, s) : hipSuccess;
  if (e == hipSuccess) e = fill(call.x, call.weight, s);
  if (e == hipSuccess && a->grad_x) {
    LinearParams p = {};
    p.Y = call.dz;
    p.ldy = call.ldz * 2;
    p.X = call.weight.at();
    p.ldx = call.weight.pitch();
    p.m = a->m;
    p.n = a->k;
    p.k = a->n;
    p.out = a->grad_x;
    p.ldo = a->k;
    p.partial = call.partial_x;
    p.slices = call.plan_x.slices;
    e = launch_two_byte(a->dtype, kGradInput, call.plan_x, p, s);
  }
  if (e == hipSuccess && a->grad_weight) {
    LinearParams p = {};
    p.Y = call.dz;
    p.ldy = call.ldz * 2;
    p.X = call.x.at();
    p.ldx = call.x.pitch();
    p.m = a->n;
    p.n = a->k;
    p.k = a->m;
    p.out = a->grad_weight;
    p.ldo = a->k;
    p.partial = call.partial_w;
    p.slices = call.plan_w.slices;
    e = launch_two_byte(a->dtype, kGradWeight, call.plan_w, p, s);
  }
  return launched(e);
}

int cumm_hip_rms_norm(const CummHipRmsNormArgs *a, void *stream) {
  if (!a) return bad("rms norm: null arguments");
  if (const char *e = norm_checked(*a)) return bad(e);
  if (a->m == 0) return CUMM_HIP_OK;
  NormParams p = {};
  p.x = a->x;
  p.residual = a->residual;
  p.weight = a->weight;
  p.out = a->out;
  p.total = a->total;
  p.codes = a->codes;
  p.scale = a->scale;
  p.inv = a->inv_rms;
  p.rows = a->m;
  p.ldx = a->ld_x;
  p.ldr = a->ld_residual;
  p.k = a->k;
  p.eps = a->eps;
  return launched(launch_norm(p, a->dtype, reinterpret_cast<hipStream_t>(stream)));
}

int64_t cumm_hip_rms_norm_backward_workspace(const CummHipRmsNormGradArgs *a) {
  if (!a || norm_grad_checked(*a)) return -1;
  return a->m == 0 || !a->grad_weight ? 0 : up((int64_t)norm_backward_blocks(a->m, a->k) * up(a->k, 16) * 4, 256);
}

int cumm_hip_rms_norm_backward(const CummHipRmsNormGradArgs *a, void *stream) {
  if (!a) return bad("rms norm backward: null arguments");
  if (const char *e = norm_grad_checked(*a)) return bad(e);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->m == 0) return launched(a->grad_weight ? launch_rows_zero(a->grad_weight, a->k, s) : hipSuccess);
  if (!a->grad_x && !a->grad_weight) return CUMM_HIP_OK;
  if (const char *e = workspace_checked(a->workspace, a->workspace_bytes, cumm_hip_rms_norm_backward_workspace(a))) return bad(e);
  NormGradParams p = {};
  p.h = a->total;
  p.weight = a->weight;
  p.grad = a->grad_out;
  p.grad_total = a->grad_total;
  p.inv = a->inv_rms;
  p.grad_in = a->grad_x;
  p.grad_weight = a->grad_weight;
  p.partial = a->grad_weight ? reinterpret_cast<float *>(a->workspace) : nullptr;
  p.rows = a->m;
  p.ldh = a->ld_total;
  p.ldg = a->ld_grad_out;
  p.ldt = a->ld_grad_total;
  p.k = a->k;
  p.pitch = (int)up(a->k, 16);
  p.blocks = norm_backward_blocks(a->m, a->k);
  return launched(launch_norm_backward(p, a->dtype == CUMM_HIP_BF16, s));
}

}  // extern "C"
