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

int check_gated(int dtype, int64_t x_stride, int64_t wg_stride, int64_t wu_stride, int act, int64_t M, int64_t N, int64_t K) {
  const int rc = check_linear(dtype, x_stride, wg_stride, act, M, N, K);
  if (rc) return rc;
  if (N >= 1 << 20) return fail(FMX_ERR_UNSUPPORTED, "N=%lld too large", (long long)N);
  return check_linear(dtype, x_stride, wu_stride, act, M, N, K);
}

// Backward workspace: dg and du beside each other, their column sums, the partial products of dx and of the
// weights' gradients (used one after the other).
struct GatedBwdWs {
  size_t dz, sums, part;
  size_t total() const { return dz + sums + part; }
};
int64_t gated_np(int64_t N) { return (N + 63) / 64 * 64; }
GatedBwdWs gated_bwd_ws(int64_t M, int64_t N, int64_t K) {
  const int64_t np = gated_np(N);
  GatedBwdWs w;
  w.dz = round256((size_t)M * (size_t)np * 4);
  w.sums = round256((size_t)fmx::gated_dz_parts(M, N) * 2 * (size_t)N * sizeof(float));
  const size_t px = fmx::linear_part_bytes(fmx::linear_plan(fmx::kLinearInput, M, K, 2 * np), M, K);
  // both weights' gradients together, or one alone
  const size_t two = fmx::linear_part_bytes(fmx::linear_plan(fmx::kLinearWeight, N, K, M, true), N, K, true);
  const size_t one = fmx::linear_part_bytes(fmx::linear_plan(fmx::kLinearWeight, N, K, M), N, K);
  const size_t pw = one > two ? one : two;
  w.part = round256(px > pw ? px : pw);
  return w;
}

int check_residual_norm(int dtype, int w_dtype, int64_t x_stride, int64_t r_stride, int64_t g_stride, double alpha, int64_t M,
                        int64_t d) {
  if (!known(dtype)) return fail(FMX_ERR_INVALID, "unknown dtype %d", dtype);
  if (w_dtype != dtype && w_dtype != FMX_DTYPE_F32)
    return fail(FMX_ERR_INVALID, "weights must be of the rows' dtype or fp32, got dtype %d", w_dtype);
  if (M < 0 || d < 1 || x_stride < 0 || r_stride < 0 || g_stride < 0)
    return fail(FMX_ERR_INVALID, "invalid sizes M=%lld d=%lld or strides", (long long)M, (long long)d);
  if (d > FMX_RESIDUAL_NORM_MAX_D)
    return fail(FMX_ERR_UNSUPPORTED, "d=%lld exceeds FMX_RESIDUAL_NORM_MAX_D=%d", (long long)d, FMX_RESIDUAL_NORM_MAX_D);
  if (!isfinite((float)alpha)) return fail(FMX_ERR_INVALID, "alpha must be finite in fp32");
  return FMX_OK;
}

int check_embedding(int dtype, int ids_bits, int64_t stride, double scale, int64_t T, int64_t V, int64_t d) {
  if (!known(dtype)) return fail(FMX_ERR_INVALID, "unknown dtype %d", dtype);
  if (ids_bits != 32 && ids_bits != 64) return fail(FMX_ERR_INVALID, "ids of %d bits, must be 32 or 64", ids_bits);
  if (T < 0 || V < 1 || d < 1 || stride < 0)
    return fail(FMX_ERR_INVALID, "invalid sizes T=%lld V=%lld d=%lld stride=%lld", (long long)T, (long long)V, (long long)d,
                (long long)stride);
  if (T > FMX_EMBEDDING_MAX_TOKENS || V > FMX_EMBEDDING_MAX_ROWS || d > FMX_MAX_D)
    return fail(FMX_ERR_UNSUPPORTED, "T=%lld V=%lld d=%lld too large", (long long)T, (long long)V, (long long)d);
  if (!isfinite((float)scale)) return fail(FMX_ERR_INVALID, "scale must be finite in fp32");
  return FMX_OK;
}

static_assert(sizeof(fmx_muon_matrix) == sizeof(fmx::MuonMatrix), "the same fields in the same order");

bool muon_sides(const fmx_muon_matrix& x) {
  const int64_t n = x.rows < x.cols ? x.rows : x.cols, m = x.rows < x.cols ? x.cols : x.rows;
  return n >= 0 && n <= FMX_MUON_MAX_SHORT && m <= FMX_MUON_MAX_LONG;
}

int check_muon(int dtype, int grad_dtype, const fmx_muon_matrix* matrices, int64_t count, int steps, double a, double b,
               double c, double eps, bool step, bool* copies) {
  if (count < 0) return fail(FMX_ERR_INVALID, "invalid count=%lld", (long long)count);
  if (steps < 1 || steps > 100) return fail(FMX_ERR_INVALID, "steps=%d must be in 1 .. 100", steps);
  if (!(eps > 0) || !isfinite(eps)) return fail(FMX_ERR_INVALID, "eps must be > 0 and finite");
  if (!(fabs(a) <= FMX_MUON_MAX_COEFFICIENT) || !(fabs(b) <= FMX_MUON_MAX_COEFFICIENT) ||
      !(fabs(c) <= FMX_MUON_MAX_COEFFICIENT))
    return fail(FMX_ERR_INVALID, "coefficients must be within +-%d", FMX_MUON_MAX_COEFFICIENT);
  if (count > 0 && !matrices) return fail(FMX_ERR_INVALID, "matrices must be non-null");
  for (int64_t i = 0; i < count; ++i) {
    const fmx_muon_matrix& x = matrices[i];
    if (x.rows < 0 || x.cols < 0)
      return fail(FMX_ERR_INVALID, "matrix %lld has %lld x %lld elements", (long long)i, (long long)x.rows, (long long)x.cols);
    if (!muon_sides(x))
      return fail(FMX_ERR_UNSUPPORTED, "matrix %lld of %lld x %lld: sides of up to %d and %d", (long long)i,
                  (long long)x.rows, (long long)x.cols, FMX_MUON_MAX_SHORT, FMX_MUON_MAX_LONG);
    if (x.rows == 0 || x.cols == 0) continue;
    if (!x.param || !x.grad || (step && !x.momentum)) return fail(FMX_ERR_INVALID, "matrix %lld: null pointer", (long long)i);
    if (!aligned(x.param, size_of(dtype)) || !aligned(x.grad, size_of(grad_dtype)) || !aligned(x.momentum, 4) ||
        !aligned(x.copy, 2))
      return fail(FMX_ERR_INVALID, "matrix %lld: pointers must be aligned to their elements", (long long)i);
    *copies |= x.copy != nullptr;
  }
  return FMX_OK;
}

int run_muon(int pd, int gd, int cd, const fmx_muon_matrix* matrices, int64_t count, fmx::MuonScalars sc, int steps, double a,
             double b, double c, double eps, void* workspace, size_t bytes, void* stream, const char* what) {
  sc.steps = steps;
  sc.a = (float)a;
  sc.b = (float)b;
  sc.c = (float)c;
  sc.eps = eps;
  const fmx::MuonMatrix* list = reinterpret_cast<const fmx::MuonMatrix*>(matrices);
  const size_t need = fmx::muon_workspace_bytes(list, count);
  if (need > 0 && (!workspace || bytes < need || !aligned(workspace, 256)))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, 256-byte aligned, %zu given", need, bytes);
  return hip_status(fmx::launch_muon(pd, gd, cd, list, count, sc, workspace, static_cast<hipStream_t>(stream)), what);
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

size_t fmx_gated_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return fmx::gated_part_bytes(fmx::gated_plan(M, N, (K + 7) / 8 * 8, false), M, N);
}

int fmx_gated(int dtype, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu,
              int64_t wu_stride, const void* bg, const void* bu, int act, int64_t M, int64_t N, int64_t K, void* y,
              int16_t* factors, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_gated(dtype, x_stride, wg_stride, wu_stride, act, M, N, K);
  if (rc) return rc;
  if (M == 0) return ok();
  if (!x || !wg || !wu || !y) return fail(FMX_ERR_INVALID, "x, wg, wu and y must be non-null");
  if (!aligned(x, 16) || !aligned(wg, 16) || !aligned(wu, 16))
    return fail(FMX_ERR_INVALID, "x, wg and wu must be 16-byte aligned");
  if (!aligned(y, 2) || !aligned(factors, 2) || !aligned(bg, 2) || !aligned(bu, 2))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  fmx::GatedArgs a = {};
  a.x = x;
  a.wg = wg;
  a.wu = wu;
  a.sx = x_stride;
  a.swg = wg_stride;
  a.swu = wu_stride;
  a.I = M;
  a.J = N;
  a.K = (K + 7) / 8 * 8;
  a.bg = bg;
  a.bu = bu;
  a.y = y;
  a.keep = factors;
  a.act = act;
  a.part = static_cast<float*>(workspace);
  const fmx::GatedPlan p = fmx::gated_plan(M, N, a.K, factors != nullptr);
  const size_t need = fmx::gated_part_bytes(p, M, N);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
  return hip_status(fmx::launch_gated(dtype == FMX_DTYPE_BF16, a, p, static_cast<hipStream_t>(stream)), "fmx_gated launch");
}

size_t fmx_gated_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return gated_bwd_ws(M, N, K).total();
}

int fmx_gated_bwd(int dtype, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu,
                  int64_t wu_stride, const void* dy, int64_t dy_stride, const int16_t* factors, int64_t M, int64_t N,
                  int64_t K, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, void* workspace, size_t workspace_bytes,
                  void* stream) {
  // x is read for the weights' gradients alone and the weights for dx; one that is missing has no stride
  const int64_t k8 = (K + 7) / 8 * 8;
  const int rc = check_gated(dtype, x ? x_stride : k8, wg ? wg_stride : k8, wu ? wu_stride : k8, FMX_ACT_NONE, M, N, K);
  if (rc) return rc;
  if (dy_stride < 0) return fail(FMX_ERR_INVALID, "dy stride must be >= 0");
  const bool weights = dwg || dwu, sums = dbg || dbu;
  if (!dx && !weights && !sums) return ok();
  if (M > 0 && ((weights && !x) || (dx && (!wg || !wu)) || !dy || !factors))
    return fail(FMX_ERR_INVALID, "x (for dwg and dwu), wg and wu (for dx), dy and factors must be non-null");
  if (!aligned(x, 16) || !aligned(wg, 16) || !aligned(wu, 16))
    return fail(FMX_ERR_INVALID, "x, wg and wu must be 16-byte aligned");
  if (!aligned(dy, 2) || !aligned(factors, 2) || !aligned(dx, 2) || !aligned(dwg, 2) || !aligned(dwu, 2) ||
      !aligned(dbg, 2) || !aligned(dbu, 2))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  const bool bf = dtype == FMX_DTYPE_BF16;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (M == 0) {  // no rows: zeros
    for (void* w : {dwg, dwu})
      if (w && e == hipSuccess) e = fmx::launch_linear_zero(w, N * K, s);
    for (void* b : {dbg, dbu})
      if (b && e == hipSuccess) e = fmx::launch_linear_zero(b, N, s);
    return hip_status(e, "fmx_gated_bwd launch");
  }
  const GatedBwdWs ws = gated_bwd_ws(M, N, K);
  if (!workspace || workspace_bytes < ws.total() || !aligned(workspace, 16))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", ws.total(), workspace_bytes);
  char* base = static_cast<char*>(workspace);
  const int64_t np = gated_np(N);
  const int parts = fmx::gated_dz_parts(M, N);
  float* column_sums = reinterpret_cast<float*>(base + ws.dz);
  fmx::GatedDzArgs z = {};
  z.dy = dy;
  z.keep = factors;
  z.dz = dx || weights ? base : nullptr;
  z.part = sums ? column_sums : nullptr;
  z.sdy = dy_stride;
  z.M = M;
  z.N = N;
  z.Np = np;
  e = fmx::launch_gated_dz(bf, z, parts, s);
  if (sums && e == hipSuccess) e = fmx::launch_join(dtype, column_sums, parts, N, N, dbg, dbu, s);
  if (e != hipSuccess) return hip_status(e, "fmx_gated_bwd launch");
  fmx::LinearArgs a = {};
  a.sa = 2 * np;
  a.part = reinterpret_cast<float*>(base + ws.dz + ws.sums);
  if (dx) {
    a.A = base;
    a.B = wg;
    a.sb = wg_stride;
    a.B2 = wu;
    a.sb2 = wu_stride;
    a.half = (int)(np / 64);
    a.kb = (int)N;
    a.I = M;
    a.J = K;
    a.K = 2 * np;
    a.y = dx;
    e = fmx::launch_linear(bf, fmx::kLinearInput, a, fmx::linear_plan(fmx::kLinearInput, M, K, 2 * np), s);
    if (e != hipSuccess) return hip_status(e, "fmx_gated_bwd launch");
    a.B2 = nullptr;
  }
  if (weights) {
    const bool both = dwg && dwu;
    a.A = base + (dwg ? 0 : np * 2);
    a.A2 = both ? base + np * 2 : nullptr;
    a.B = x;
    a.sb = x_stride;
    a.I = N;
    a.J = K;
    a.K = M;
    a.y = dwg ? dwg : dwu;
    a.y2 = both ? dwu : nullptr;
    e = fmx::launch_linear(bf, fmx::kLinearWeight, a, fmx::linear_plan(fmx::kLinearWeight, N, K, M, both), s);
  }
  return hip_status(e, "fmx_gated_bwd launch");
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

int fmx_residual_norm(int dtype, const void* x, int64_t x_stride, const void* residual, int64_t r_stride, const void* gate,
                      int64_t g_stride, int w_dtype, const void* weight, const void* bias, int post, const void* post_weight,
                      const void* post_bias, const void* scale, double alpha, int rms, double eps, int64_t M, int64_t d,
                      void* h, void* y, float* stats, void* stream) {
  const int rc = check_residual_norm(dtype, w_dtype, x_stride, r_stride, gate ? g_stride : 0, alpha, M, d);
  if (rc) return rc;
  if (!(eps >= 0)) return fail(FMX_ERR_INVALID, "eps must be >= 0");
  if (!post && (post_weight || post_bias)) return fail(FMX_ERR_INVALID, "weights of a norm of x that is not wanted");
  if (M == 0) return ok();
  if (!x || !residual || !h || !y) return fail(FMX_ERR_INVALID, "x, residual, h and y must be non-null");
  const int es = size_of(dtype), ws = size_of(w_dtype);
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(gate, es) || !aligned(h, es) || !aligned(y, es) ||
      !aligned(weight, ws) || !aligned(bias, ws) || !aligned(post_weight, ws) || !aligned(post_bias, ws) ||
      !aligned(scale, ws))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  if (!aligned(stats, 16)) return fail(FMX_ERR_INVALID, "stats must be 16-byte aligned");
  fmx::ResidualNormArgs a = {};
  a.x = x;
  a.r = residual;
  a.gate = gate;
  a.w = weight;
  a.b = bias;
  a.pw = post_weight;
  a.pb = post_bias;
  a.scale = scale;
  a.h = h;
  a.y = y;
  a.stats = stats;
  a.sx = x_stride;
  a.sr = r_stride;
  a.sg = g_stride;
  a.M = M;
  a.d = (int)d;
  a.w32 = w_dtype == FMX_DTYPE_F32;
  a.rms = rms != 0;
  a.post = post != 0;
  a.alpha = (float)alpha;
  a.eps = (float)eps;
  return hip_status(fmx::launch_residual_norm_fwd(dtype, a, static_cast<hipStream_t>(stream)), "fmx_residual_norm launch");
}

size_t fmx_residual_norm_bwd_workspace_bytes(int64_t M, int64_t d) {
  if (M < 1 || d < 1 || d > FMX_RESIDUAL_NORM_MAX_D) return 0;
  return (size_t)fmx::residual_norm_parts(M, (int)d) * 5 * (size_t)d * sizeof(float);
}

int fmx_residual_norm_bwd(int dtype, const void* x, int64_t x_stride, const void* residual, int64_t r_stride,
                          const void* gate, int64_t g_stride, int w_dtype, const void* weight, int post,
                          const void* post_weight, const void* post_bias, const void* scale, double alpha, int rms,
                          const float* stats, const void* dh, int64_t dh_stride, const void* dy, int64_t dy_stride, int64_t M,
                          int64_t d, void* dx, void* dr, void* dgate, void* dw, void* db, void* dscale, void* dpw, void* dpb,
                          void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_residual_norm(dtype, w_dtype, x_stride, r_stride, gate ? g_stride : 0, alpha, M, d);
  if (rc) return rc;
  if ((dh && dh_stride < 0) || (dy && dy_stride < 0)) return fail(FMX_ERR_INVALID, "strides must be >= 0");
  if (!post && (dpw || dpb)) return fail(FMX_ERR_INVALID, "gradients of a norm of x that is not there");
  if (dgate && !gate) return fail(FMX_ERR_INVALID, "a gradient of a gate that is not there");
  const bool any = dx || dr || dgate || dw || db || dscale || dpw || dpb;
  if (!any) return ok();
  if (M > 0 && (!x || !residual || !stats || (!dh && !dy)))
    return fail(FMX_ERR_INVALID, "x, residual, stats and one of dh and dy must be non-null");
  if ((dw || db) && M > 0 && !dy) return fail(FMX_ERR_INVALID, "dw and db come of dy");
  const int es = size_of(dtype), ws = size_of(w_dtype);
  for (const void* p : {x, residual, gate, dh, dy, (const void*)dx, (const void*)dr, (const void*)dgate})
    if (!aligned(p, es)) return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  for (const void* p : {weight, post_weight, post_bias, scale, (const void*)dw, (const void*)db, (const void*)dscale,
                        (const void*)dpw, (const void*)dpb})
    if (!aligned(p, ws)) return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  if (!aligned(stats, 16)) return fail(FMX_ERR_INVALID, "stats must be 16-byte aligned");
  fmx::ResidualNormArgs a = {};
  a.sums[0] = dw;
  a.sums[1] = db;
  a.sums[2] = dscale;
  a.sums[3] = dpw;
  a.sums[4] = dpb;
  for (void* s : a.sums) a.wanted += s != nullptr;
  const size_t need = a.wanted ? fmx_residual_norm_bwd_workspace_bytes(M, d) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
  a.x = x;
  a.r = residual;
  a.gate = gate;
  a.w = weight;
  a.pw = post_weight;
  a.pb = post_bias;
  a.scale = scale;
  a.stats = const_cast<float*>(stats);
  a.dh = dh;
  a.dy = dy;
  a.dx = dx;
  a.dr = dr;
  a.dgate = dgate;
  a.part = a.wanted ? static_cast<float*>(workspace) : nullptr;
  a.sx = x_stride;
  a.sr = r_stride;
  a.sg = g_stride;
  a.sdh = dh_stride;
  a.sdy = dy_stride;
  a.M = M;
  a.d = (int)d;
  a.w32 = w_dtype == FMX_DTYPE_F32;
  a.rms = rms != 0;
  a.post = post != 0;
  a.alpha = (float)alpha;
  return hip_status(fmx::launch_residual_norm_bwd(dtype, a, static_cast<hipStream_t>(stream)),
                    "fmx_residual_norm_bwd launch");
}

int fmx_embedding(int dtype, const void* ids, int ids_bits, const void* w, int64_t w_stride, double scale, int64_t T, int64_t V,
                  int64_t d, void* y, void* stream) {
  const int rc = check_embedding(dtype, ids_bits, w_stride, scale, T, V, d);
  if (rc) return rc;
  if (T == 0) return ok();
  if (!ids || !w || !y) return fail(FMX_ERR_INVALID, "ids, w and y must be non-null");
  if (!aligned(ids, ids_bits / 8) || !aligned(w, size_of(dtype)) || !aligned(y, size_of(dtype)))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  fmx::EmbeddingArgs a = {};
  a.ids = ids;
  a.ids64 = ids_bits == 64;
  a.w = w;
  a.sw = w_stride;
  a.out = y;
  a.T = T;
  a.V = V;
  a.d = (int)d;
  a.scale = (float)scale;
  return hip_status(fmx::launch_embedding(dtype, a, static_cast<hipStream_t>(stream)), "fmx_embedding launch");
}

size_t fmx_embedding_bwd_workspace_bytes(int dtype, int64_t T, int64_t V, int64_t d) {
  if (!known(dtype) || T < 0 || V < 1 || d < 1 || T > FMX_EMBEDDING_MAX_TOKENS || V > FMX_EMBEDDING_MAX_ROWS || d > FMX_MAX_D)
    return 0;
  return fmx::embedding_workspace_bytes(dtype, T, V, d);
}

int fmx_embedding_bwd(int dtype, const void* ids, int ids_bits, const void* dy, int64_t dy_stride, double scale,
                      int64_t padding_id, int64_t T, int64_t V, int64_t d, void* dw, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const int rc = check_embedding(dtype, ids_bits, dy_stride, scale, T, V, d);
  if (rc) return rc;
  if ((T > 0 && (!ids || !dy)) || !dw) return fail(FMX_ERR_INVALID, "ids, dy and dw must be non-null");
  if (!aligned(ids, ids_bits / 8) || !aligned(dy, size_of(dtype)) || !aligned(dw, size_of(dtype)))
    return fail(FMX_ERR_INVALID, "pointers must be aligned to their elements");
  const size_t need = fmx_embedding_bwd_workspace_bytes(dtype, T, V, d);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return fail(FMX_ERR_WORKSPACE, "workspace of %zu bytes required, 256-byte aligned, %zu given", need, workspace_bytes);
  fmx::EmbeddingArgs a = {};
  a.ids = ids;
  a.ids64 = ids_bits == 64;
  a.dy = dy;
  a.sdy = dy_stride;
  a.out = dw;
  a.T = T;
  a.V = V;
  a.d = (int)d;
  a.padding = padding_id;
  a.scale = (float)scale;
  return hip_status(fmx::launch_embedding_bwd(dtype, a, workspace, static_cast<hipStream_t>(stream)),
                    "fmx_embedding_bwd launch");
}

size_t fmx_muon_workspace_bytes(const fmx_muon_matrix* matrices, int64_t count) {
  if (!matrices || count < 1) return 0;
  for (int64_t i = 0; i < count; ++i)
    if (!muon_sides(matrices[i])) return 0;
  return fmx::muon_workspace_bytes(reinterpret_cast<const fmx::MuonMatrix*>(matrices), count);
}

int fmx_muon(int param_dtype, int grad_dtype, int copy_dtype, const fmx_muon_matrix* matrices, int64_t count, double lr,
             double momentum, int nesterov, double weight_decay, int steps, double a, double b, double c, double eps,
             int match_rms, const float* grad_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!known(param_dtype) || !known(grad_dtype))
    return fail(FMX_ERR_INVALID, "unknown dtype %d or %d", param_dtype, grad_dtype);
  if (!(lr >= 0) || !(weight_decay >= 0) || !(momentum >= 0 && momentum < 1))
    return fail(FMX_ERR_INVALID, "lr and weight_decay must be >= 0, momentum in [0, 1)");
  bool copies = false;
  const int rc = check_muon(param_dtype, grad_dtype, matrices, count, steps, a, b, c, eps, true, &copies);
  if (rc) return rc;
  if (copies && (param_dtype != FMX_DTYPE_F32 || (copy_dtype != FMX_DTYPE_F16 && copy_dtype != FMX_DTYPE_BF16)))
    return fail(FMX_ERR_INVALID, "copies are fp16 or bf16, of fp32 parameters");
  if (!copies) copy_dtype = grad_dtype != FMX_DTYPE_F32 ? grad_dtype : FMX_DTYPE_BF16;
  if (grad_dtype != FMX_DTYPE_F32 && grad_dtype != param_dtype &&
      !(param_dtype == FMX_DTYPE_F32 && grad_dtype == copy_dtype))
    return fail(FMX_ERR_INVALID, "gradients must be fp32 or of the parameters' (or their copies') dtype");
  fmx::MuonScalars sc = {};
  sc.lr = lr;
  sc.mu = (float)momentum;
  sc.omu = (float)(1.0 - momentum);
  sc.keep = (float)(1.0 - lr * weight_decay);
  sc.nesterov = nesterov != 0;
  sc.by_rms = match_rms != 0;
  sc.apply = 1;
  sc.grad_scale = grad_scale;
  return run_muon(param_dtype, grad_dtype, copy_dtype, matrices, count, sc, steps, a, b, c, eps, workspace, workspace_bytes,
                  stream, "fmx_muon launch");
}

int fmx_orthogonalize(int out_dtype, int dtype, const fmx_muon_matrix* matrices, int64_t count, int steps, double a, double b,
                      double c, double eps, void* workspace, size_t workspace_bytes, void* stream) {
  if (!known(out_dtype) || !known(dtype)) return fail(FMX_ERR_INVALID, "unknown dtype %d or %d", out_dtype, dtype);
  bool copies = false;
  const int rc = check_muon(out_dtype, dtype, matrices, count, steps, a, b, c, eps, false, &copies);
  if (rc) return rc;
  fmx::MuonScalars sc = {};
  return run_muon(out_dtype, dtype, FMX_DTYPE_BF16, matrices, count, sc, steps, a, b, c, eps, workspace, workspace_bytes,
                  stream, "fmx_orthogonalize launch");
}

}  // extern "C"
