// Layer norm over rows of d elements, forward and backward.
//
//   mu = mean x, s = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) s, y = xh w + b
//   dx = s (wdy - mean(wdy) - xh mean(wdy xh)), wdy = w dy
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// Bound by HBM: the forward reads and writes every element once, the backward
// reads x and dy and writes dx. A row lives in registers between its sums and
// its output: up to 16 elements a lane in one, two, four or eight waves (at 32
// the backward's sums, weights and two rows spill), and only rows of more than
// 8192 (forward: 16384) elements are read again for each sum. A workgroup's eight
// waves walk the rows in strides of the launch, so each holds its columns' w and
// b, and in the backward their dw and db in float32, in registers for all of its
// rows; the next row is loaded while this one is summed. The variance is that of centred
// values (a second sum over registers, no second read), so a row's mean takes
// no digits from it.
//
// Weight gradients: a workgroup adds its waves' sums in LDS in the waves' order and writes
// one row of partial sums; a second kernel adds those rows in a fixed order. No
// atomics, so the same inputs give the same bits.
#include "fmx_device.h"
#include "fmx_layers.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

template <typename T, int V>
struct __attribute__((aligned(sizeof(T) * V > 16 ? 16 : sizeof(T) * V))) Pack {
  T v[V];
};

constexpr int kWaves = 8;  // of a workgroup
constexpr int kThreads = kWaves * 64;

// Sum of a and of b over the NW waves that share a row (1: the wave alone), in every lane.
template <int NW>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int wave) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = a;
      red[2 * wave + 1] = b;
    }
    __syncthreads();
    const float* mine = red + 2 * (wave & -NW);
    a = 0.0f;
    b = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      a += mine[2 * i];
      b += mine[2 * i + 1];
    }
  }
}
template <int NW>
__device__ __forceinline__ float row_sum(float a, float* red, int wave) {
  a = wave_sum(a);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) red[wave] = a;
    __syncthreads();
    const float* mine = red + (wave & -NW);
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) a += mine[i];
  }
  return a;
}

// Where a lane's elements lie: chunk j of V elements at column
// ((j * NW + sub) * 64 + lane) * V, sub the wave's place among the NW of its row.
template <typename T, int V, int NV, int NW>
struct Cols {
  int col[NV];
  bool in[NV];
  __device__ __forceinline__ Cols(int wave, int lane, int d) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      col[j] = ((j * NW + wave % NW) * 64 + lane) * V;
      in[j] = col[j] < d;  // V > 1: d is a multiple of V
    }
  }
  // a row's elements; zeros past it, and everywhere without a row
  __device__ __forceinline__ void load(Pack<T, V> (&x)[NV], const T* row, bool have) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (in[j] && have) {
        x[j] = *reinterpret_cast<const Pack<T, V>*>(row + col[j]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[j].v[i] = T(0.0f);
      }
    }
  }
  // w or b as float32, `other` where there is none or past the row; 16-byte aligned where V > 1
  template <typename W>
  __device__ __forceinline__ void weights_of(float (&o)[NV][V], const W* w, float other) const {
    Pack<W, V> p[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (in[j]) p[j] = *reinterpret_cast<const Pack<W, V>*>(w + col[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = in[j] ? (float)p[j].v[i] : other;
  }
  __device__ __forceinline__ void weights(float (&o)[NV][V], const void* w, int w32, float other) const {
    if (!w) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) o[j][i] = other;
    } else if (w32) {
      weights_of(o, static_cast<const float*>(w), other);
    } else {
      weights_of(o, static_cast<const T*>(w), other);
    }
  }
};

template <typename T, int V, int NV, int NW>
__global__ void __launch_bounds__(kThreads) norm_fwd_kernel(NormArgs a) {
  constexpr int NG = kWaves / NW;  // rows of a workgroup at a time
  __shared__ float red[2][kWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Cols<T, V, NV, NW> c(wave, lane, a.d);
  const float inv = 1.0f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * NG;
  const T* x0 = static_cast<const T*>(a.x);
  T* y0 = static_cast<T*>(a.y);
  Pack<T, V> x[NV], next[NV];
  int64_t row = (int64_t)blockIdx.x * NG + wave / NW;
  c.load(x, x0 + row * a.sx, row < a.M);
  float w[NV][V], b[NV][V];
  c.weights(w, a.w, a.w32, 1.0f);
  c.weights(b, a.b, a.w32, 0.0f);
  // base, and so the number of barriers, is the same for all rows of the workgroup
  for (int64_t base = (int64_t)blockIdx.x * NG; base < a.M; base += step, row += step) {
    c.load(next, x0 + (row + step) * a.sx, row + step < a.M);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += (float)x[j].v[i];
    const float mu = row_sum<NW>(sum, red[0], wave) * inv;
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = (float)x[j].v[i] - mu;
        sq += c.in[j] ? e * e : 0.0f;
      }
    const float rs = 1.0f / sqrtf(row_sum<NW>(sq, red[1], wave) * inv + a.eps);
    if (row < a.M) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!c.in[j]) continue;
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = (T)(((float)x[j].v[i] - mu) * rs * w[j][i] + b[j][i]);
        *reinterpret_cast<Pack<T, V>*>(y0 + row * a.d + c.col[j]) = o;
      }
      if (a.mean && lane == 0 && wave % NW == 0) {
        a.mean[row] = mu;
        a.rstd[row] = rs;
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j] = next[j];
  }
}

template <typename T, int V, int NV, int NW>
__global__ void __launch_bounds__(kThreads) norm_bwd_kernel(NormArgs a) {
  constexpr int NG = kWaves / NW;
  constexpr int W = 64 * V * NV * NW;  // columns that the registers of a row hold
  __shared__ float red[2][2 * kWaves];
  __shared__ float fold[NG > 1 ? 2 * W : 1];  // the workgroup's rows' sums of dw and db meet here
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Cols<T, V, NV, NW> c(wave, lane, a.d);
  float w[NV][V], dw[NV][V], db[NV][V];
  c.weights(w, a.w, a.w32, 1.0f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[j][i] = 0.0f;
      db[j][i] = 0.0f;
    }
  const float inv = 1.0f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * NG;
  const T* x0 = static_cast<const T*>(a.x);
  const T* dy0 = static_cast<const T*>(a.dy);
  T* dx0 = static_cast<T*>(a.y);
  Pack<T, V> x[NV], g[NV], nx[NV], ng[NV];
  int64_t row = (int64_t)blockIdx.x * NG + wave / NW;
  c.load(x, x0 + row * a.sx, row < a.M);
  c.load(g, dy0 + row * a.sdy, row < a.M);
  float mu = row < a.M ? a.mean[row] : 0.0f, rs = row < a.M ? a.rstd[row] : 0.0f;
  int par = 0;
  for (int64_t base = (int64_t)blockIdx.x * NG; base < a.M; base += step, row += step) {
    const bool more = row + step < a.M;
    c.load(nx, x0 + (row + step) * a.sx, more);
    c.load(ng, dy0 + (row + step) * a.sdy, more);
    const float nmu = more ? a.mean[row + step] : 0.0f, nrs = more ? a.rstd[row + step] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // past the row, and without one, x, dy and so every term are zero times a finite number:
        // xh there is -mu rs, which only a row that is not finite itself makes otherwise
        const float xh = ((float)x[j].v[i] - mu) * rs, dy = (float)g[j].v[i], wdy = dy * w[j][i];
        s1 += wdy;
        s2 += c.in[j] ? wdy * xh : 0.0f;
        dw[j][i] += dy * xh;
        db[j][i] += dy;
      }
    if (a.y) {
      row_sum2<NW>(s1, s2, red[par], wave);
      par ^= 1;
      const float c1 = s1 * inv, c2 = s2 * inv;
      if (row < a.M) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!c.in[j]) continue;
          Pack<T, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float xh = ((float)x[j].v[i] - mu) * rs;
            o.v[i] = (T)(rs * ((float)g[j].v[i] * w[j][i] - c1 - xh * c2));
          }
          *reinterpret_cast<Pack<T, V>*>(dx0 + row * a.d + c.col[j]) = o;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = nx[j];
      g[j] = ng[j];
    }
    mu = nmu;
    rs = nrs;
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.d;
  if constexpr (NG > 1) {
    for (int k = 0; k < NG; ++k) {
      if (wave / NW == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int at = c.col[j] + i;
            fold[at] = k ? fold[at] + dw[j][i] : dw[j][i];
            fold[W + at] = k ? fold[W + at] + db[j][i] : db[j][i];
          }
      }
      __syncthreads();
    }
    for (int at = threadIdx.x; at < a.d; at += kThreads) {
      part[at] = fold[at];
      part[a.d + at] = fold[W + at];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c.in[j]) {
          part[c.col[j] + i] = dw[j][i];
          part[a.d + c.col[j] + i] = db[j][i];
        }
  }
}

// Rows of any width, a workgroup each, read once for every sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_fwd_wide_kernel(NormArgs a) {
  __shared__ float red[2][kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = 1.0f / (float)a.d;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    T* y = static_cast<T*>(a.y) + row * a.d;
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.d; k += kThreads) sum += (float)x[k];
    const float mu = row_sum<kWaves>(sum, red[0], wave) * inv;
    float sq = 0.0f;
    for (int k = threadIdx.x; k < a.d; k += kThreads) sq += ((float)x[k] - mu) * ((float)x[k] - mu);
    const float rs = 1.0f / sqrtf(row_sum<kWaves>(sq, red[1], wave) * inv + a.eps);
    for (int k = threadIdx.x; k < a.d; k += kThreads) {
      const float w = !a.w ? 1.0f : a.w32 ? static_cast<const float*>(a.w)[k] : (float)static_cast<const T*>(a.w)[k];
      const float b = !a.b ? 0.0f : a.w32 ? static_cast<const float*>(a.b)[k] : (float)static_cast<const T*>(a.b)[k];
      y[k] = (T)(((float)x[k] - mu) * rs * w + b);
    }
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
  }
}

// dx of rows of any width, a workgroup each.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_dx_wide_kernel(NormArgs a) {
  __shared__ float red[2][2 * kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = 1.0f / (float)a.d;
  int par = 0;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.sdy;
    T* dx = static_cast<T*>(a.y) + row * a.d;
    const float mu = a.mean[row], rs = a.rstd[row];
    auto wdy = [&](int k) {
      const float w = !a.w ? 1.0f : a.w32 ? static_cast<const float*>(a.w)[k] : (float)static_cast<const T*>(a.w)[k];
      return w * (float)dy[k];
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (int k = threadIdx.x; k < a.d; k += kThreads) {
      s1 += wdy(k);
      s2 += wdy(k) * (((float)x[k] - mu) * rs);
    }
    row_sum2<kWaves>(s1, s2, red[par], wave);
    par ^= 1;
    for (int k = threadIdx.x; k < a.d; k += kThreads)
      dx[k] = (T)(rs * (wdy(k) - s1 * inv - ((float)x[k] - mu) * rs * (s2 * inv)));
  }
}

// Partial dw and db of rows of any width: a lane a column, a workgroup row (y) a stretch of rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_dw_wide_kernel(NormArgs a) {
  const int k = blockIdx.x * 256 + threadIdx.x;
  if (k >= a.d) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    const float dy = (float)static_cast<const T*>(a.dy)[row * a.sdy + k];
    dw += dy * (((float)static_cast<const T*>(a.x)[row * a.sx + k] - a.mean[row]) * a.rstd[row]);
    db += dy;
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.d;
  part[k] = dw;
  part[a.d + k] = db;
}

// Sums of the columns of `parts` rows of n0 + n1 values, the first n0 to out0, the others to out1.
// 16 columns a workgroup, its threads 64 rows at a time: 512 rows of 2048 columns 11.2 us with 64 columns
// (32 workgroups, 32 rows a wave one after the other), 4.4 with 16.
template <typename O>
__global__ void __launch_bounds__(1024) join_kernel(const float* part, int parts, int64_t n0, int64_t n1, O* out0,
                                                    O* out1) {
  __shared__ float sums[64][17];
  const int c = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int64_t k = (int64_t)blockIdx.x * 16 + c, n = n0 + n1;
  float s = 0.0f;
  if (k < n) {
#pragma unroll 4
    for (int p = group; p < parts; p += 64) s += part[p * n + k];
  }
  sums[group][c] = s;
  __syncthreads();
#pragma unroll
  for (int half = 32; half >= 4; half /= 2) {  // to four sums a column
    if (group < half) sums[group][c] += sums[group + half][c];
    __syncthreads();
  }
  if (group == 0 && k < n) {
    s = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
    O* out = k < n0 ? out0 : out1;
    if (out) out[k < n0 ? k : k - n0] = (O)s;
  }
}

// Waves of a row: as few as hold it with 16 elements a lane; 0: none do, the row is read again for
// each sum. The forward's registers also hold 32 a lane.
constexpr int kMaxE = 16;
int waves_of(int d, bool bwd) {
  for (int nw = 1; nw <= kWaves; nw *= 2)
    if (d <= 64 * nw * kMaxE) return nw;
  return !bwd && d <= 64 * kWaves * 2 * kMaxE ? kWaves : 0;
}

// Workgroups for M rows, `group` at a time: as many as run at once (per_cu on each compute unit), so that
// all of them share the rows evenly. 65536 x 1024 bf16 forward, of whose workgroups a unit holds three:
// four a unit 66 us, three 56.
int grid_of(int64_t M, int group, int per_cu) {
  const int64_t want = (M + group - 1) / group, most = (int64_t)layer_cus() * per_cu;
  return (int)(want < most ? want : most);
}

// Workgroups of this kernel that a compute unit holds.
int held(const void* kernel) {
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, 0) != hipSuccess || n < 1) n = 1;
  return n;
}

// Backward workgroups write their partial sums once each: two a unit at most.
constexpr int kBwdPerCu = 2;

template <typename T, int V, int E, int NW>
int run(const NormArgs& a, bool bwd, hipStream_t s) {
  constexpr int group = kWaves / NW;
  if constexpr (E <= kMaxE) {
    if (bwd) {
      static const int n = held(reinterpret_cast<const void*>(norm_bwd_kernel<T, V, E / V, NW>));
      const int grid = grid_of(a.M, group, n < kBwdPerCu ? n : kBwdPerCu);
      norm_bwd_kernel<T, V, E / V, NW><<<grid, kThreads, 0, s>>>(a);
      return grid;
    }
  }
  static const int n = held(reinterpret_cast<const void*>(norm_fwd_kernel<T, V, E / V, NW>));
  const int grid = grid_of(a.M, group, n);
  norm_fwd_kernel<T, V, E / V, NW><<<grid, kThreads, 0, s>>>(a);
  return grid;
}

template <typename T, int V, int NW>
int run_nw(const NormArgs& a, bool bwd, hipStream_t s) {
  const int e = (a.d + 64 * NW - 1) / (64 * NW);  // elements a lane
  if constexpr (NW == 1) {
    if (e <= 4 && V <= 4) return run<T, V, V <= 4 ? 4 : 8, NW>(a, bwd, s);
    if (e <= 8) return run<T, V, 8, NW>(a, bwd, s);
  }
  if (V <= 4 && e <= 12) return run<T, V, V <= 4 ? 12 : 16, NW>(a, bwd, s);
  if constexpr (NW == kWaves) {
    if (e > 16) return run<T, V, 32, NW>(a, false, s);
  }
  return run<T, V, 16, NW>(a, bwd, s);
}

template <typename T, int V>
int run_v(const NormArgs& a, int nw, bool bwd, hipStream_t s) {
  switch (nw) {
    case 1: return run_nw<T, V, 1>(a, bwd, s);
    case 2: return run_nw<T, V, 2>(a, bwd, s);
    case 4: return run_nw<T, V, 4>(a, bwd, s);
    default: return run_nw<T, V, 8>(a, bwd, s);
  }
}

constexpr int kWideParts = 64;  // stretches of rows whose weight gradients the wide kernel sums

// *parts: the rows of partial sums written, of the backward
template <typename T>
hipError_t launch(const NormArgs& a, bool vec, bool bwd, int* parts, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int nw = waves_of(a.d, bwd);
  if (nw) {
    *parts = vec ? run_v<T, V>(a, nw, bwd, s) : run_v<T, 1>(a, nw, bwd, s);
  } else if (!bwd) {
    norm_fwd_wide_kernel<T><<<grid_of(a.M, 1, 4), kThreads, 0, s>>>(a);
  } else {
    if (a.y) norm_dx_wide_kernel<T><<<grid_of(a.M, 1, 4), kThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    *parts = a.M < kWideParts ? (int)a.M : kWideParts;
    if (a.part) norm_dw_wide_kernel<T><<<dim3((a.d + 255) / 256, *parts), 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_kind(int kind, const NormArgs& a, bool vec, bool bwd, int* parts, hipStream_t s) {
  if (kind == FMX_DTYPE_F32) return launch<float>(a, vec, bwd, parts, s);
  if (kind == FMX_DTYPE_BF16) return launch<__bf16>(a, vec, bwd, parts, s);
  return launch<_Float16>(a, vec, bwd, parts, s);
}

}  // namespace

int norm_parts(int64_t M, int d) {
  const int nw = waves_of(d, true);
  return nw ? grid_of(M, kWaves / nw, kBwdPerCu) : (int)(M < kWideParts ? M : kWideParts);
}

hipError_t launch_norm_fwd(int kind, const NormArgs& a, bool vec, hipStream_t s) {
  int parts;
  return launch_kind(kind, a, vec, false, &parts, s);
}
hipError_t launch_norm_bwd(int kind, const NormArgs& a, bool vec, int* parts, hipStream_t s) {
  return launch_kind(kind, a, vec, true, parts, s);
}

hipError_t launch_join(int out_kind, const float* part, int parts, int64_t n0, int64_t n1, void* out0, void* out1,
                       hipStream_t s) {
  const unsigned grid = (unsigned)((n0 + n1 + 15) / 16);
  if (out_kind == FMX_DTYPE_F32)
    join_kernel<<<grid, 1024, 0, s>>>(part, parts, n0, n1, static_cast<float*>(out0), static_cast<float*>(out1));
  else if (out_kind == FMX_DTYPE_BF16)
    join_kernel<<<grid, 1024, 0, s>>>(part, parts, n0, n1, static_cast<__bf16*>(out0), static_cast<__bf16*>(out1));
  else
    join_kernel<<<grid, 1024, 0, s>>>(part, parts, n0, n1, static_cast<_Float16*>(out0), static_cast<_Float16*>(out1));
  return hipGetLastError();
}

}  // namespace fmx
