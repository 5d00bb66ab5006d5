// C ABI of the trained layers: argument checks and workspace sizes. Declarations
// and the contract live in include/fmx.h.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/fmx.h"
#include "fmx_layers.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return fmx::report(code, buf);
}

int ok() { return fmx::report(FMX_OK, nullptr); }

int hip_status(hipError_t e, const char* what) {
  return e == hipSuccess ? ok() : fail(FMX_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool known(int dtype) { return dtype == FMX_DTYPE_F16 || dtype == FMX_DTYPE_BF16 || dtype == FMX_DTYPE_F32; }
int size_of(int dtype) { return dtype == FMX_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

int check_norm(int dtype, int w_dtype, int64_t x_stride, int64_t M, int64_t d) {
  if (!known(dtype)) return fail(FMX_ERR_INVALID, "unknown dtype %d", dtype);
  if (w_dtype != dtype && w_dtype != FMX_DTYPE_F32)
    return fail(FMX_ERR_INVALID, "weights must be of the rows' dtype or fp32, got dtype %d", w_dtype);
  if (M < 0 || d < 1 || x_stride < 0)
    return fail(FMX_ERR_INVALID, "invalid sizes M=%lld d=%lld stride=%lld", (long long)M, (long long)d,
                (long long)x_stride);
  if (d > FMX_MAX_D) return fail(FMX_ERR_UNSUPPORTED, "d=%lld exceeds FMX_MAX_D=%d", (long long)d, FMX_MAX_D);
  return FMX_OK;
}

int check_linear(int dtype, int64_t x_stride, int64_t w_stride, int act, int64_t M, int64_t N, int64_t K) {
  if (dtype != FMX_DTYPE_F16 && dtype != FMX_DTYPE_BF16) return fail(FMX_ERR_INVALID, "unknown dtype %d", dtype);
  if (act < FMX_ACT_NONE || act > FMX_ACT_SILU) return fail(FMX_ERR_INVALID, "unknown activation %d", act);
  if (M < 0 || N < 1 || K < 1)
    return fail(FMX_ERR_INVALID, "invalid sizes M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (M > FMX_LINEAR_MAX_ROWS || N >= 1 << 24 || K >= 1 << 24)
    return fail(FMX_ERR_UNSUPPORTED, "M=%lld N=%lld K=%lld too large", (long long)M, (long long)N, (long long)K);
  const int64_t k8 = (K + 7) / 8 * 8;
  if (x_stride < k8 || (x_stride & 7) || w_stride < k8 || (w_stride & 7))
    return fail(FMX_ERR_INVALID, "row strides %lld and %lld must be >= K rounded up to 8 and multiples of 8",
                (long long)x_stride, (long long)w_stride);
  if (x_stride >= 1 << 22 || w_stride >= 1 << 22)
    return fail(FMX_ERR_UNSUPPORTED, "row strides %lld and %lld must be < 2^22", (long long)x_stride,
                (long long)w_stride);
  return FMX_OK;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Backward workspace: dz, the column sums, the partial products of dx and of dw (used one after
// the other).
struct LinearBwdWs {
  size_t dz, sums, part;
  size_t total() const { return dz + sums + part; }
};
LinearBwdWs linear_bwd_ws(int64_t M, int64_t N, int64_t K) {
  const int64_t n8 = (N + 7) / 8 * 8;
  LinearBwdWs w;
  w.dz = round256((size_t)M * (size_t)n8 * 2);
  const fmx::LinearPlan plan_w = fmx::linear_plan(fmx::kLinearWeight, N, K, M);
  const int parts = fmx::linear_dz_parts(M, N);
  w.sums = round256((size_t)(parts > plan_w.splits ? parts : plan_w.splits) * (size_t)N * sizeof(float));
  const size_t px = fmx::linear_part_bytes(fmx::linear_plan(fmx::kLinearInput, M, K, n8), M, K);
  const size_t pw = fmx::linear_part_bytes(plan_w, N, K);
  w.part = round256(px > pw ? px : pw);
  return w;
}

}  // namespace

extern "C" {

size_t fmx_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return fmx::linear_part_bytes(fmx::linear_plan(fmx::kLinearForward, M, N, (K + 7) / 8 * 8), M, N);
}

int fmx_linear(int dtype, const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias,
               const void* residual, int64_t r_stride, int act, int64_t M, int64_t N, int64_t K, void* y, int16_t* slope,
               void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_linear(dtype, x_stride, w_stride, act, M, N, K);
  if (rc) return rc;
  if (residual && r_stride < 0) return fail(FMX_ERR_INVALID, "residual stride must be >= 0");
  if (M == 0) return ok();
  if (!x || !w || !y) return fail(FMX_ERR_INVALID, "x, w and y must be non-null");
  if (!aligned(x, 16) || !aligned(w, 16)) return fail(FMX_ERR_INVALID, "x and w must be 16-byte aligned");
  if (!aligned(y, 2) || !aligned(slope, 2) || !aligned(bias, 2) || !aligned(residual, 2))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  fmx::LinearArgs a = {};
  a.A = x;
  a.B = w;
  a.sa = x_stride;
  a.sb = w_stride;
  a.I = M;
  a.J = N;
  a.K = (K + 7) / 8 * 8;
  a.y = y;
  a.slope = act == FMX_ACT_NONE ? nullptr : slope;
  a.bias = bias;
  a.res = residual;
  a.sres = r_stride;
  a.act = act;
  a.part = static_cast<float*>(workspace);
  const fmx::LinearPlan p = fmx::linear_plan(fmx::kLinearForward, M, N, a.K);
  const size_t need = fmx::linear_part_bytes(p, M, N);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
  return hip_status(fmx::launch_linear(dtype == FMX_DTYPE_BF16, fmx::kLinearForward, a, p,
                                       static_cast<hipStream_t>(stream)),
                    "fmx_linear launch");
}

size_t fmx_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return linear_bwd_ws(M, N, K).total();
}

int fmx_linear_bwd(int dtype, const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* dy,
                   int64_t dy_stride, const int16_t* slope, int act, int64_t M, int64_t N, int64_t K, void* dx, void* dw,
                   void* db, void* workspace, size_t workspace_bytes, void* stream) {
  // x is read for dw alone and w for dx; one that is missing has no stride
  const int64_t k8 = (K + 7) / 8 * 8;
  const int rc = check_linear(dtype, x ? x_stride : k8, w ? w_stride : k8, act, M, N, K);
  if (rc) return rc;
  if (dy_stride < 0) return fail(FMX_ERR_INVALID, "dy stride must be >= 0");
  if (!dx && !dw && !db) return ok();
  if (M > 0 && ((dw && !x) || (dx && !w) || !dy || (act != FMX_ACT_NONE && !slope)))
    return fail(FMX_ERR_INVALID, "x (for dw), w (for dx), dy and (with an activation) slope must be non-null");
  if (!aligned(x, 16) || !aligned(w, 16)) return fail(FMX_ERR_INVALID, "x and w must be 16-byte aligned");
  if (!aligned(dy, 2) || !aligned(slope, 2) || !aligned(dx, 2) || !aligned(dw, 2) || !aligned(db, 2))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  const bool bf = dtype == FMX_DTYPE_BF16;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (M == 0) {  // no rows: zeros
    hipError_t e = hipSuccess;
    if (dw) e = fmx::launch_linear_zero(dw, N * K, s);
    if (db && e == hipSuccess) e = fmx::launch_linear_zero(db, N, s);
    return hip_status(e, "fmx_linear_bwd launch");
  }
  const LinearBwdWs ws = linear_bwd_ws(M, N, K);
  if (!workspace || workspace_bytes < ws.total() || !aligned(workspace, 16))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", ws.total(), workspace_bytes);
  char* base = static_cast<char*>(workspace);
  const int64_t n8 = (N + 7) / 8 * 8;
  // dy serves as dz where it is one already and its rows can be read as an operand
  const bool as_is = act == FMX_ACT_NONE && N % 8 == 0 && dy_stride % 8 == 0 && dy_stride >= N &&
                     dy_stride < 1 << 22 && aligned(dy, 16);
  const bool make = !as_is && (dx || dw);
  const fmx::LinearPlan plan_w = fmx::linear_plan(fmx::kLinearWeight, N, K, M);
  // its columns' sums come with the dw product where dy needs no pass of its own
  const bool beside = as_is && dw && db && fmx::linear_sums_columns(plan_w);
  const bool later = dw && db && plan_w.splits > 1;  // added up by the launch that joins dw's parts
  const int parts = beside ? plan_w.splits : fmx::linear_dz_parts(M, N);
  float* sums = reinterpret_cast<float*>(base + ws.dz);
  hipError_t e = hipSuccess;
  if (make || (db && !beside)) {
    fmx::DzArgs a = {};
    a.dy = dy;
    a.slope = act == FMX_ACT_NONE ? nullptr : slope;
    a.dz = make ? base : nullptr;
    a.part = db ? sums : nullptr;
    a.sdy = dy_stride;
    a.M = M;
    a.N = N;
    a.Np = n8;
    e = fmx::launch_linear_dz(bf, a, parts, s);
    if (db && !later && e == hipSuccess) e = fmx::launch_join(dtype, sums, parts, N, 0, db, nullptr, s);
    if (e != hipSuccess) return hip_status(e, "fmx_linear_bwd launch");
  }
  fmx::LinearArgs a = {};
  a.A = as_is ? dy : base;
  a.sa = as_is ? dy_stride : n8;
  a.part = reinterpret_cast<float*>(base + ws.dz + ws.sums);
  if (dx) {
    a.B = w;
    a.sb = w_stride;
    a.I = M;
    a.J = K;
    a.K = N;
    a.y = dx;
    e = fmx::launch_linear(bf, fmx::kLinearInput, a, fmx::linear_plan(fmx::kLinearInput, M, K, n8), s);
    if (e != hipSuccess) return hip_status(e, "fmx_linear_bwd launch");
  }
  if (dw) {
    a.B = x;
    a.sb = x_stride;
    a.I = N;
    a.J = K;
    a.K = M;
    a.y = dw;
    a.db_part = sums;
    a.db_beside = beside;
    a.db_parts = parts;
    a.db = later ? db : nullptr;
    e = fmx::launch_linear(bf, fmx::kLinearWeight, a, plan_w, s);
    if (beside && !later && e == hipSuccess) e = fmx::launch_join(dtype, sums, parts, N, 0, db, nullptr, s);
  }
  return hip_status(e, "fmx_linear_bwd launch");
}

int fmx_layer_norm(int dtype, const void* x, int64_t x_stride, int w_dtype, const void* weight, const void* bias,
                   int64_t M, int64_t d, double eps, void* y, float* mean, float* rstd, void* stream) {
  const int rc = check_norm(dtype, w_dtype, x_stride, M, d);
  if (rc) return rc;
  if (!(eps >= 0)) return fail(FMX_ERR_INVALID, "eps must be >= 0");
  if (!mean != !rstd) return fail(FMX_ERR_INVALID, "mean and rstd go together");
  if (M == 0) return ok();
  if (!x || !y) return fail(FMX_ERR_INVALID, "x and y must be non-null");
  const int es = size_of(dtype), ws = size_of(w_dtype), V = 16 / es;
  if (!aligned(x, es) || !aligned(y, es) || !aligned(weight, ws) || !aligned(bias, ws))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  fmx::NormArgs a = {};
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.sx = x_stride;
  a.M = M;
  a.d = (int)d;
  a.w32 = w_dtype == FMX_DTYPE_F32;
  a.eps = (float)eps;
  const bool vec = d % V == 0 && x_stride % V == 0 && aligned(x, 16) && aligned(y, 16) &&
                   aligned(weight, 16) && aligned(bias, 16);
  return hip_status(fmx::launch_norm_fwd(dtype, a, vec, static_cast<hipStream_t>(stream)), "fmx_layer_norm launch");
}

size_t fmx_layer_norm_bwd_workspace_bytes(int64_t M, int64_t d) {
  if (M < 1 || d < 1 || d > FMX_MAX_D) return 0;
  return (size_t)fmx::norm_parts(M, (int)d) * 2 * (size_t)d * sizeof(float);
}

int fmx_layer_norm_bwd(int dtype, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int w_dtype,
                       const void* weight, const float* mean, const float* rstd, int64_t M, int64_t d, void* dx,
                       void* dw, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_norm(dtype, w_dtype, x_stride < dy_stride ? x_stride : dy_stride, M, d);
  if (rc) return rc;
  const int es = size_of(dtype), ws = size_of(w_dtype), V = 16 / es;
  const bool sums = dw || db;
  if (M > 0 && (dx || sums) && (!x || !dy || !mean || !rstd))
    return fail(FMX_ERR_INVALID, "x, dy, mean and rstd must be non-null");
  if (!aligned(x, es) || !aligned(dy, es) || !aligned(dx, es) || !aligned(weight, ws) || !aligned(dw, ws) ||
      !aligned(db, ws))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  const size_t need = sums ? fmx_layer_norm_bwd_workspace_bytes(M, d) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int parts = 0;  // no rows: zeros
  if (M > 0 && (dx || sums)) {
    fmx::NormArgs a = {};
    a.x = x;
    a.dy = dy;
    a.w = weight;
    a.y = dx;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    a.sx = x_stride;
    a.sdy = dy_stride;
    a.M = M;
    a.d = (int)d;
    a.w32 = w_dtype == FMX_DTYPE_F32;
    const bool vec = d % V == 0 && x_stride % V == 0 && dy_stride % V == 0 && aligned(x, 16) && aligned(dy, 16) &&
                     aligned(dx, 16) && aligned(weight, 16);
    const hipError_t e = fmx::launch_norm_bwd(dtype, a, vec, &parts, s);
    if (e != hipSuccess) return hip_status(e, "fmx_layer_norm_bwd launch");
  }
  if (sums) {
    return hip_status(fmx::launch_join(w_dtype, static_cast<const float*>(workspace), parts, d, d, dw, db, s),
                      "fmx_layer_norm_bwd launch");
  }
  return ok();
}

int fmx_adamw(int param_dtype, int grad_dtype, int copy_dtype, int state_bits, const fmx_adamw_tensor* tensors,
              int64_t count, int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
              const float* grad_scale, void* stream) {
  if (!known(param_dtype) || !known(grad_dtype))
    return fail(FMX_ERR_INVALID, "unknown dtype %d or %d", param_dtype, grad_dtype);
  if (state_bits != 8 && state_bits != 32) return fail(FMX_ERR_INVALID, "state_bits=%d must be 8 or 32", state_bits);
  if (count < 0 || step < 1)
    return fail(FMX_ERR_INVALID, "invalid count=%lld or step=%lld", (long long)count, (long long)step);
  if (!(lr >= 0) || !(eps >= 0) || !(weight_decay >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1))
    return fail(FMX_ERR_INVALID, "lr, eps and weight_decay must be >= 0, betas in [0, 1)");
  if (count > 0 && !tensors) return fail(FMX_ERR_INVALID, "tensors must be non-null");
  bool copies = false;
  const int ps = size_of(param_dtype), gs = size_of(grad_dtype), ss = state_bits == 8 ? 1 : 4;
  for (int64_t i = 0; i < count; ++i) {
    const fmx_adamw_tensor& t = tensors[i];
    if (t.n < 0) return fail(FMX_ERR_INVALID, "tensor %lld has %lld elements", (long long)i, (long long)t.n);
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
        (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return fail(FMX_ERR_INVALID, "tensor %lld: null pointer", (long long)i);
    if (!aligned(t.param, ps) || !aligned(t.grad, gs) || !aligned(t.exp_avg, ss) || !aligned(t.exp_avg_sq, ss) ||
        !aligned(t.exp_avg_scale, 4) || !aligned(t.exp_avg_sq_scale, 4) || !aligned(t.copy, 2))
      return fail(FMX_ERR_INVALID, "tensor %lld: pointers must be aligned to their elements", (long long)i);
    copies |= t.copy != nullptr;
  }
  if (copies && (param_dtype != FMX_DTYPE_F32 || (copy_dtype != FMX_DTYPE_F16 && copy_dtype != FMX_DTYPE_BF16)))
    return fail(FMX_ERR_INVALID, "copies are fp16 or bf16, of fp32 parameters");
  if (!copies) copy_dtype = grad_dtype != FMX_DTYPE_F32 ? grad_dtype : FMX_DTYPE_BF16;
  if (grad_dtype != FMX_DTYPE_F32 && grad_dtype != param_dtype &&
      !(param_dtype == FMX_DTYPE_F32 && grad_dtype == copy_dtype))
    return fail(FMX_ERR_INVALID, "gradients must be fp32 or of the parameters' (or their copies') dtype");
  static_assert(sizeof(fmx_adamw_tensor) == sizeof(fmx::AdamWTensor), "the same fields in the same order");
  fmx::AdamWScalars sc;
  sc.beta1 = (float)beta1;
  sc.omb1 = (float)(1.0 - beta1);
  sc.beta2 = (float)beta2;
  sc.omb2 = (float)(1.0 - beta2);
  sc.keep = (float)(1.0 - lr * weight_decay);
  sc.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  sc.eps = (float)eps;
  sc.rate = (float)(lr / (1.0 - pow(beta1, (double)step)));
  sc.grad_scale = grad_scale;
  return hip_status(fmx::launch_adamw(param_dtype, grad_dtype, copy_dtype, state_bits,
                                      reinterpret_cast<const fmx::AdamWTensor*>(tensors), count, sc,
                                      static_cast<hipStream_t>(stream)),
                    "fmx_adamw launch");
}

int fmx_adamw_decode(int second, const void* codes, const float* scales, int64_t n, float* out, void* stream) {
  if (n < 0) return fail(FMX_ERR_INVALID, "n=%lld must be >= 0", (long long)n);
  if (n == 0) return ok();
  if (!codes || !scales || !out) return fail(FMX_ERR_INVALID, "codes, scales and out must be non-null");
  if (!aligned(scales, 4) || !aligned(out, 4)) return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  return hip_status(fmx::launch_adamw_decode(codes, second != 0, scales, n, out, static_cast<hipStream_t>(stream)),
                    "fmx_adamw_decode launch");
}

}  // extern "C"
