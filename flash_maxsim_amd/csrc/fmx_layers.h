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
int norm_parts(int64_t M, int d);  // rows of NormArgs::part
hipError_t launch_norm_fwd(int kind, const NormArgs& a, bool vec, hipStream_t s);
hipError_t launch_norm_bwd(int kind, const NormArgs& a, bool vec, hipStream_t s);
// out0[c] = sum over parts of part[p][0][c], out1 likewise; either may be null.
hipError_t launch_norm_join(int out_kind, const float* part, int parts, int d, void* out0, void* out1, hipStream_t s);

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

}  // namespace fmx
