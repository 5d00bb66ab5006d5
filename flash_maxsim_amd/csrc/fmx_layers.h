// Launchers and argument structs of the trained layers around MaxSim: layer
// norm, linear and the AdamW step. The C ABI in fmx_layers_api.hip validates
// arguments; the launchers pick the template instance and enqueue it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmx {

// Sets the calling thread's error message (fmx_last_error) and returns code
// (fmx_api.hip); a null message clears it.
int report(int code, const char* message);
// Compute units of the current device.
int layer_cus();

// ---- layer norm (fmx_norm.hip) ----

struct NormArgs {
  const void* x;    // [M, d], row stride sx
  const void* dy;   // backward: [M, d], row stride sdy
  const void* w;    // [d], or null (ones)
  const void* b;    // [d], or null (zeros); forward only
  void* y;          // forward: y, backward: dx; [M, d] contiguous; backward: may be null
  float* mean;      // [M]; forward: written unless null
  float* rstd;      // [M]
  float* part;      // backward: partial sums [parts][2][d], or null (no weight gradients)
  int64_t sx, sdy;
  int64_t M;
  int d;
  int w32;          // w and b are float32, else of x's type
  float eps;
};

// kind: FMX_DTYPE_*
int norm_parts(int64_t M, int d);  // rows of NormArgs::part at most
hipError_t launch_norm_fwd(int kind, const NormArgs& a, bool vec, hipStream_t s);
// *parts: the rows of NormArgs::part written
hipError_t launch_norm_bwd(int kind, const NormArgs& a, bool vec, int* parts, hipStream_t s);
// Sums over `parts` rows of n0 + n1 float32 values: the first n0 columns to out0, the others to out1, in
// out_kind's type; either may be null. No rows: zeros. 64 threads a column: fewer than 2^26 columns.
hipError_t launch_join(int out_kind, const float* part, int parts, int64_t n0, int64_t n1, void* out0, void* out1,
                       hipStream_t s);

// ---- AdamW (fmx_adamw.hip) ----

struct AdamWTensor {
  void* param;
  const void* grad;
  void* m;       // float32, or int8 codes
  void* v;       // float32, or uint8 codes of its root
  float* ms;     // 8 bits: a scale per block of 256
  float* vs;
  void* copy;    // 16-bit copy of the new parameters, or null
  int64_t n;
};

struct AdamWScalars {
  float beta1, omb1, beta2, omb2;  // omb: 1 - beta
  float keep;                      // 1 - lr * weight decay
  float root;                      // 1 / sqrt(1 - beta2^step)
  float eps;
  float rate;                      // lr / (1 - beta1^step)
  const float* grad_scale;         // one value, or null
};

hipError_t launch_adamw(int pkind, int gkind, int ckind, int bits, const AdamWTensor* t, int64_t count,
                        const AdamWScalars& sc, hipStream_t s);
hipError_t launch_adamw_decode(const void* codes, bool second, const float* scales, int64_t n, float* out, hipStream_t s);

// ---- linear (fmx_linear.hip) ----

enum LinearForm { kLinearForward, kLinearInput, kLinearWeight };  // y, dx, dw
enum LinearTile { kTile64, kTile128, kTile128Deep, kTile256, kFewRows };  // deep: four stages in LDS, not two

// C[I, J] = sum over k < K of A(i, k) B(j, k); see fmx_linear.hip for the operands of each form.
struct LinearArgs {
  const void* A;
  const void* B;
  int64_t sa, sb;         // row strides in memory, multiples of 8
  int64_t I, J, K;        // K: a multiple of 8 where it runs along rows
  int64_t Jr;             // B's columns or rows that exist (set by launch_linear)
  void* y;                // [I, J] 16-bit, contiguous
  void* slope;            // forward: act's slopes in their 16-bit code, [I, J]; or null
  const void* bias;       // forward: [J], or null
  const void* res;        // forward: [I, J], row stride sres, or null
  int64_t sres;
  float* part;            // splits > 1: [splits][I][Jp]
  float* db_part;         // dw: sums over k of A's columns, [db_parts][I]
  int db_beside;          // dw: this product writes them, [splits][I]
  int db_parts;
  void* db;               // dw, splits > 1: their totals, by the second kernel; or null
  int64_t Jp;
  int64_t ti, tj;         // tiles
  int64_t split_k, band;
  int splits;
  int act;
};

struct LinearPlan {
  int tile;
  int size;               // of the tile
  int splits;
  int64_t ti, tj, split_k, band;
};
LinearPlan linear_plan(LinearForm form, int64_t I, int64_t J, int64_t K);
size_t linear_part_bytes(const LinearPlan& p, int64_t I, int64_t J);
// Whether the dw product of this plan adds up its A's columns beside it (its registers hold no more at 256 x 256).
inline bool linear_sums_columns(const LinearPlan& p) { return p.tile != kTile256; }
hipError_t launch_linear(bool bf16, LinearForm form, LinearArgs a, const LinearPlan& p, hipStream_t s);

struct DzArgs {
  const void* dy;         // [M, N], row stride sdy
  const void* slope;      // [M, N] contiguous, or null (no activation)
  void* dz;               // [M, Np] 16-bit, or null
  float* part;            // [parts][N] column sums, or null
  int64_t sdy, M, N, Np;  // Np: N rounded up to 8
  int lanes;              // of a row, a power of two; set by launch_linear_dz
};
int linear_dz_parts(int64_t M, int64_t N);
hipError_t launch_linear_dz(bool bf16, DzArgs a, int parts, hipStream_t s);
hipError_t launch_linear_zero(void* out, int64_t n, hipStream_t s);  // n > 0 zeros of 16 bits

}  // namespace fmx
