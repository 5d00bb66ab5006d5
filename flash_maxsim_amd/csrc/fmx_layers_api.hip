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

}  // namespace

extern "C" {

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
  const bool vec = d % V == 0 && x_stride % V == 0 && aligned(x, 16) && aligned(y, 16);
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
                     aligned(dx, 16);
    const hipError_t e = fmx::launch_norm_bwd(dtype, a, vec, s);
    if (e != hipSuccess) return hip_status(e, "fmx_layer_norm_bwd launch");
  }
  if (sums) {
    const int parts = M > 0 ? fmx::norm_parts(M, (int)d) : 0;  // no rows: zeros
    return hip_status(fmx::launch_norm_join(w_dtype, static_cast<const float*>(workspace), parts, (int)d, dw, db, s),
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
