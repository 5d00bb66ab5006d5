// Orthogonalised updates (as the Muon optimiser makes them), many matrices in one launch.
//
//   m = mu m + (1 - mu) g,   u = (1 - mu) g + mu m  (or m),   X = u / |u|_F, its shorter side first
//   steps times:  A = X X^T,  B = a I + b A + c A^2,  X = B X
//   p = p (1 - lr decay) - rate X
//
// Every singular value s of X goes to a s + b s^3 + c s^5, towards 1 from anywhere; a is large, so that small
// ones grow quickly: five steps with a = 3.44 multiply them by up to 485, and with them whatever error lies in
// their directions. Products run on fp16 MFMA with float32 sums. Where an error comes in, and what it costs
// (relative distance of the result from 64 bits; matrices of falling, flat and few singular values):
//   X rounded to fp16        1.2e-3 to 4e-2: its rounding lies in all directions and grows 485-fold with them
//   (bf16 for everything     1e-2 to 3e-1)
//   X as a pair of fp16      2e-4 to 3.5e-3: the linear term a X takes both, the products only the upper half. What
//                            the lower half would add there is (B - a I) times it, which is small but where X is large
//   a I within B             4e-4 to 2.3e-3: the upper half's linear term is part of its product, exact but for the
//                            rounding of B's diagonal, which scales rows and does not grow
// so X lies in memory as two fp16 arrays, of which the lower one is read and written by the epilogue alone (X = B X_upper +
// a X_lower): no product more. The last form saves the epilogue X's upper half (24 matrices of 1024 x 4096: 302 us a
// launch, 364 with it read; B's diagonal's rest as a product of its own in the loop 448). X is held times
// 2^8, A and B times 2^10: their small elements stay clear of fp16's subnormal ones.
//
// A and B are symmetric: tiles on and below the diagonal are computed, and a tile that lies below leaves LDS
// twice, the second time through transposing reads. Matrices taller than wide are transposed when X is made, and the
// last product's epilogue, which moves the parameters, transposes back.
//
// A launch walks the tiles of up to kMost matrices of any shapes, from a table in its arguments.
#include <math.h>

#include "fmx_device.h"
#include "fmx_layers.h"
#include "fmx_product.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

constexpr float kX = 256.0f, kA = 1024.0f;  // what X, and A and B, are held times
constexpr int kMost = 40;                   // matrices of a launch: their table fits a kernel's arguments
constexpr int kPad = 64;                    // X's sides in the workspace are multiples of this, the rest is zeros
constexpr int kChunk = 8192;                // elements whose squares one workgroup adds up

struct Entry {
  void* param;          // or the orthogonalised result
  const void* grad;
  float* momentum;      // or null: u is the gradient itself
  void* copy;
  int64_t at;           // of its part of the workspace, bytes
  int32_t rows, cols;   // of the parameter
  int32_t n, m;         // of X, padded: n the shorter side
  float rate;
  int32_t unused;
};

struct Table {
  char* ws;
  const float* grad_scale;
  double eps;
  float mu, omu, keep;          // omu: 1 - mu
  float a, b, c;
  int nesterov, apply;          // apply: parameters move; else the result is written
  uint32_t total;               // workgroups
  int count, from;              // from: which of the two X is read
  uint32_t first[kMost];        // an entry's first workgroup of the launch; past the last one: all ones
  Entry e[kMost];
};
static_assert(sizeof(Table) <= 4096, "kernel arguments");

// An entry's arrays in the workspace, in order: X twice, its lower halves, A, B (16-bit), the sums of squares (doubles).
__host__ __device__ inline int64_t x_bytes(const Entry& e) { return (int64_t)e.n * e.m * 2; }
__host__ __device__ inline int64_t a_bytes(const Entry& e) { return (int64_t)e.n * e.n * 2; }
__device__ __forceinline__ uint16_t* x_of(const Table& t, const Entry& e, int which) {
  return reinterpret_cast<uint16_t*>(t.ws + e.at + which * x_bytes(e));
}
__device__ __forceinline__ uint16_t* low_of(const Table& t, const Entry& e) { return x_of(t, e, 2); }
__device__ __forceinline__ uint16_t* a_of(const Table& t, const Entry& e) {
  return reinterpret_cast<uint16_t*>(t.ws + e.at + 3 * x_bytes(e));
}
__device__ __forceinline__ uint16_t* b_of(const Table& t, const Entry& e) {
  return reinterpret_cast<uint16_t*>(t.ws + e.at + 3 * x_bytes(e) + a_bytes(e));
}
__device__ __forceinline__ double* squares_of(const Table& t, const Entry& e) {
  return reinterpret_cast<double*>(t.ws + e.at + 3 * x_bytes(e) + 2 * a_bytes(e));
}

// The entry that workgroup `id` works for: the last one whose first workgroup is not past it. One load for all: a search
// waits for the arguments' memory once for every step (a step over four small matrices, 17 launches, 102 us by a search, 97).
__device__ __forceinline__ int entry_of(const Table& t, uint32_t id) {
  const int lane = threadIdx.x & 63;
  const uint32_t first = t.first[lane < kMost ? lane : kMost - 1];
  return __builtin_popcountll(__ballot(lane < kMost && first <= id)) - 1;
}

// 8 consecutive values from element `at` of a row-major array, `left` of them there (at least 1; none: zeros).
template <int KIND>
__device__ __forceinline__ void load8(float (&v)[8], const void* base, int64_t at, int left) {
  if constexpr (KIND == FMX_DTYPE_F32) {
    const float* p = static_cast<const float*>(base) + at;
    if (left >= 8) {
      __builtin_memcpy(v, p, 32);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : 0.0f;
    }
  } else {
    if (left > 0) {
      load16(v, base, at, left, KIND == FMX_DTYPE_BF16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    }
  }
}
template <int KIND>
__device__ __forceinline__ void store8(void* base, int64_t at, int left, const float (&v)[8]) {
  if constexpr (KIND == FMX_DTYPE_F32) {
    float* p = static_cast<float*>(base) + at;
    if (left >= 8) {
      __builtin_memcpy(p, v, 32);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) p[k] = v[k];
    }
  } else {
    store16(base, at, left, v, KIND == FMX_DTYPE_BF16);
  }
}

// u of 8 elements from the gradient and the (new) momentum.
__device__ __forceinline__ void direction(float (&u)[8], const float (&g)[8], const float (&m)[8], const Table& t,
                                          bool momentum, float scale) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float x = g[k] * scale;
    u[k] = !momentum ? x : t.nesterov ? t.omu * x + t.mu * m[k] : m[k];
  }
}

// The new momentum, and the sum of u's squares over each chunk (double: no gradient is too large or small to square).
template <int G>
__global__ void __launch_bounds__(256) muon_momentum_kernel(Table t) {
  __shared__ double sums[256];
  const int at = entry_of(t, blockIdx.x);
  const Entry& e = t.e[at];
  const uint32_t chunk = blockIdx.x - t.first[at];
  const int64_t size = (int64_t)e.rows * e.cols;
  const float scale = t.grad_scale ? *t.grad_scale : 1.0f;
  double sum = 0.0;
#pragma unroll
  for (int v = 0; v < kChunk / 2048; ++v) {
    const int64_t from = (int64_t)chunk * kChunk + v * 2048 + threadIdx.x * 8;
    if (from >= size) break;
    const int left = size - from < 8 ? (int)(size - from) : 8;
    float g[8], m[8], u[8];
    load8<G>(g, e.grad, from, left);
    if (e.momentum) {
      load8<FMX_DTYPE_F32>(m, e.momentum, from, left);
#pragma unroll
      for (int k = 0; k < 8; ++k) m[k] = t.mu * m[k] + t.omu * (g[k] * scale);
      store8<FMX_DTYPE_F32>(e.momentum, from, left, m);
    }
    direction(u, g, m, t, e.momentum != nullptr, scale);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += k < left ? (double)u[k] * (double)u[k] : 0.0;
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int half = 128; half > 0; half /= 2) {
    if ((int)threadIdx.x < half) sums[threadIdx.x] += sums[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x == 0) squares_of(t, e)[chunk] = sums[0];
}

// X of 64 x 64 elements: u over its norm, in two halves, transposed where the parameter is taller than wide.
template <int G>
__global__ void __launch_bounds__(256) muon_start_kernel(Table t) {
  __shared__ double sums[256];
  __shared__ float tile[64][65];
  const int at = entry_of(t, blockIdx.x);
  const Entry& e = t.e[at];
  const uint32_t id = blockIdx.x - t.first[at], tj = (uint32_t)e.m / 64, ti = id / tj;
  const int i0 = (int)ti * 64, j0 = (int)(id - ti * tj) * 64;
  const int64_t size = (int64_t)e.rows * e.cols, chunks = (size + kChunk - 1) / kChunk;
  double sum = 0.0;
  for (int64_t k = threadIdx.x; k < chunks; k += 256) sum += squares_of(t, e)[k];
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int half = 128; half > 0; half /= 2) {
    if ((int)threadIdx.x < half) sums[threadIdx.x] += sums[threadIdx.x + half];
    __syncthreads();
  }
  const double norm = sqrt(sums[0]);
  const double by = (double)kX / (norm <= t.eps ? t.eps : norm);  // a norm that is NaN stays so
  const float scale = t.grad_scale ? *t.grad_scale : 1.0f;
  const bool tall = e.rows > e.cols;
  const int row = threadIdx.x >> 2, part = (threadIdx.x & 3) * 16;
  // the tile's rows as the parameter has them: of i, or of j
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  float x[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + row, c = c0 + part + 8 * h;
    const int left = r < e.rows ? (e.cols - c < 8 ? e.cols - c : 8) : 0;
    float g[8], m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = m[k] = 0.0f;
    if (left > 0) {
      const int64_t at = (int64_t)r * e.cols + c;
      load8<G>(g, e.grad, at, left);
      if (e.momentum) load8<FMX_DTYPE_F32>(m, e.momentum, at, left);
    }
    direction(x[h], g, m, t, e.momentum != nullptr, scale);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[h][k] = k < left ? (float)((double)x[h][k] * by) : 0.0f;
  }
  if (tall) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 8; ++k) tile[part + 8 * h + k][row] = x[h][k];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 8; ++k) x[h][k] = tile[row][part + 8 * h + k];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t at = (int64_t)(i0 + row) * e.m + j0 + part + 8 * h;
    const u32x4_t hi = pack8(x[h], false);
    float up[8];
    unpack8(up, hi, false);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[h][k] -= up[k];
    store_raw(x_of(t, e, 0), at, 8, hi);
    store_raw(low_of(t, e), at, 8, pack8(x[h], false));
  }
}

// ---- the products ----

enum Form { kGram, kPolynomial, kNext, kLast };  // A, B, X, and the parameters by the last X

// The last product's values of 8 elements of one of the parameter's rows.
template <int P>
__device__ __forceinline__ void move8(const Table& t, const Entry& e, int64_t at, int left, float (&x)[8], int copy_bf) {
  if (t.apply) {
    float p[8];
    load8<P>(p, e.param, at, left);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = p[k] * t.keep - e.rate * x[k];
  }
  store8<P>(e.param, at, left, x);
  if (P == FMX_DTYPE_F32 && e.copy) store16(e.copy, at, left, x, copy_bf);
}

// P: the parameters' type (kLast)
template <int FORM, int P, int WI, int WJ, int FI, int FJ, int NS>
__global__ void __launch_bounds__(WI* WJ * 64) muon_kernel(Table t, int copy_bf) {
  constexpr bool SYM = FORM == kGram || FORM == kPolynomial, BMAJ = !SYM;
  constexpr int TI = WI * FI * 16, TJ = WJ * FJ * 16, NT = WI * WJ * 64;
  constexpr int BYTES = (TI + TJ) * BK * 2;
  static_assert(TI == TJ, "square tiles: the symmetric products' tiles lie on or below the diagonal");
  using SideA = Side<false, false, TI, NT>;
  using SideB = Side<BMAJ, !BMAJ, TJ, NT>;
  constexpr int LOADS = SideA::kLoads + SideB::kLoads;
  __shared__ __attribute__((aligned(1024))) unsigned char lds0[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds1[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds2[NS > 2 ? BYTES : 16];
  __shared__ __attribute__((aligned(1024))) unsigned char lds3[NS > 2 ? BYTES : 16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave % WI, wj = wave / WI;
  // workgroups go to the eight XCDs in turn; each XCD takes a run of consecutive tiles
  uint32_t id = blockIdx.x;
  {
    const uint32_t per = t.total / 8, x = id & 7, rest = t.total & 7;
    id = (id >> 3) + x * per + (x < rest ? x : rest);
  }
  const int at = entry_of(t, id);
  const Entry& e = t.e[at];
  id -= t.first[at];
  uint32_t row, col;
  if constexpr (SYM) {  // row r of the triangle begins at r (r + 1) / 2
    row = (uint32_t)((sqrtf(8.0f * (float)id + 1.0f) - 1.0f) * 0.5f);
    while (row * (row + 1) / 2 > id) --row;
    while ((row + 1) * (row + 2) / 2 <= id) ++row;
    col = id - row * (row + 1) / 2;
  } else {  // the rows of a column of tiles, which read the same columns of X, one after the other
    const uint32_t ti = (uint32_t)(e.n + TI - 1) / TI;
    col = id / ti;
    row = id - col * ti;
  }
  const int64_t i0 = (int64_t)row * TI, j0 = (int64_t)col * TJ;
  const int depth = FORM == kGram ? e.m : e.n, nit = depth / BK;
  const int64_t width = SYM ? e.n : e.m;  // columns of the result
  const uint16_t *A, *B;
  if constexpr (FORM == kGram) {
    A = B = x_of(t, e, t.from);
  } else if constexpr (FORM == kPolynomial) {
    A = B = a_of(t, e);
  } else {
    A = b_of(t, e);
    B = x_of(t, e, t.from);
  }
  const SideA sa(A, FORM == kGram ? e.m : e.n, i0, e.n, 0, tid);
  const SideB sb(B, FORM == kPolynomial ? e.n : e.m, j0, width, 0, tid);
  const Frags<false, false, TI> fa(wi * FI * 16, lane);
  const Frags<BMAJ, !BMAJ, TJ> fb(wj * FJ * 16, lane);

  f32x4_t acc[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto buffer = [&](auto s) -> unsigned char* {
    constexpr int S = decltype(s)::value % NS;
    if constexpr (S == 0) return lds0;
    if constexpr (S == 1) return lds1;
    if constexpr (S == 2) return lds2;
    return lds3;
  };
  auto issue = [&](unsigned char* lds, int it) __attribute__((always_inline)) {
    const int left = depth - it * BK;
    sa.issue(lds, it, left, wave);
    sb.issue(lds + TI * BK * 2, it, left, wave);
  };
  u32x4_t va[2][FI], vb[2][FJ];
  auto read = [&](auto set, const unsigned char* lds, int kk) __attribute__((always_inline)) {
    constexpr int Z = decltype(set)::value;
#pragma unroll
    for (int y = 0; y < FJ; ++y) vb[Z][y] = fb.read(lds + TI * BK * 2, y, kk);
#pragma unroll
    for (int x = 0; x < FI; ++x) va[Z][x] = fa.read(lds, x, kk);
  };
  auto multiply = [&](auto set) __attribute__((always_inline)) {
    constexpr int Z = decltype(set)::value;
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y) acc[x][y] = mfma16x16x32<false>(vb[Z][y], va[Z][x], acc[x][y]);
  };
  run_stages<NS, LOADS, FJ*(BMAJ ? 2 : 1) + FI, FI * FJ>(nit, buffer, issue, read, multiply, [](auto) {});

  // A lane's results: row c of each i fragment, and of a pair of j fragments 8 columns, from column `of` of the pair's 32 on.
  const int c = lane & 15, g = lane >> 4;
  const int of = BMAJ ? (g & 1) * 16 + (g >> 1) * 8 : 8 * g;
  auto pair = [&](int x, int y, float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = acc[x][y][k];
      v[4 + k] = acc[x][y + 1][k];
      if constexpr (BMAJ) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v[k]),
                                                        __builtin_bit_cast(uint32_t, v[4 + k]), false, false);
        const uint32_t r0 = r[0], r1 = r[1];
        v[k] = __builtin_bit_cast(float, r0);
        v[4 + k] = __builtin_bit_cast(float, r1);
      }
    }
  };
  stage_barrier();  // LDS is free: nothing is loaded into it or read from it any more
  constexpr int ROW = FJ * 32;  // bytes of a wave's 16-bit row
  unsigned char* mine = (wave < WI * WJ / 2 ? lds0 : lds1) + (wave % (WI * WJ / 2)) * (BYTES / (WI * WJ / 2));
  static_assert(BYTES / (WI * WJ / 2) >= FI * 16 * ROW && BYTES / (WI * WJ / 2) >= FJ * 16 * 17 * 4, "a wave's block");
  const int64_t iw = i0 + wi * FI * 16, jw = j0 + wj * FJ * 16;
  if (jw >= width) return;  // sides are multiples of 64 and a wave's block begins at one of FJ * 16

  // 16-bit rows of the block in LDS, 16 bytes at a time, and from there to memory as whole lines
  auto spot = [&](int r, int ch) __attribute__((always_inline)) { return mine + r * ROW + ((ch ^ (r & (ROW / 16 - 1))) << 4); };
  auto put = [&](int x, int ch, const u32x4_t& w) __attribute__((always_inline)) {
    *reinterpret_cast<u32x4_t*>(spot(x * 16 + c, ch)) = w;
  };
  auto flush = [&](int x, uint16_t* out) __attribute__((always_inline)) {
    constexpr int CH = ROW / 16;  // of a row
#pragma unroll
    for (int h = 0; h < 16 * CH / 64; ++h) {
      const int r = x * 16 + h * (64 / CH) + lane / CH, ch = lane % CH;
      store_raw(out, (iw + r) * width + jw + ch * 8, 8, *reinterpret_cast<const u32x4_t*>(spot(r, ch)));
    }
  };

  if constexpr (SYM) {
    uint16_t* out = FORM == kGram ? a_of(t, e) : b_of(t, e);
    const uint16_t* in = a_of(t, e);
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      if (iw + x * 16 >= e.n) break;
#pragma unroll
      for (int y = 0; y < FJ; y += 2) {
        float v[8];
        pair(x, y, v);
        const int64_t at = (iw + x * 16 + c) * e.n + jw + y * 16 + of;
        if constexpr (FORM == kGram) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] *= kA / (kX * kX);
        } else {
          float w[8];
          load16(w, in, at, 8, false);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = t.b * w[k] + (t.c / kA) * v[k];
          const int64_t off = iw + x * 16 + c - (jw + y * 16 + of);  // of the diagonal among the 8
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += k == off ? t.a * kA : 0.0f;
        }
        put(x, y * 2 + of / 8, pack8(v, false));
      }
      flush(x, out);
    }
    if (row == col) return;  // the whole tile is there
    // column j of the block: its 8 rows i .. i + 7 a lane, read as two 4 x 16 blocks turned round
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    const int q = c >> 2, s = c & 3;
#pragma unroll
    for (int x = 0; x < FI; x += 2) {  // 32 rows: 8 for each group of 16 lanes
      if (iw + x * 16 >= e.n) break;
#pragma unroll
      for (int y = 0; y < FJ; ++y) {
        const int r = x * 16 + g * 8 + q, ch = 2 * y + (s >> 1);
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(spot(r, ch) + 8 * (s & 1)));
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(spot(r + 4, ch) + 8 * (s & 1)));
        const u32x2_t l = __builtin_bit_cast(u32x2_t, lo), h = __builtin_bit_cast(u32x2_t, hi);
        store_raw(out, (jw + y * 16 + c) * e.n + iw + x * 16 + g * 8, 8, u32x4_t{l[0], l[1], h[0], h[1]});
      }
    }
  } else {
    uint16_t* xl = low_of(t, e);
    const bool tall = e.rows > e.cols;
    float* turn = reinterpret_cast<float*>(mine);  // kLast of a tall parameter: [FJ * 16][17], a 16-row block turned round
    // everything that is read, before the first store: loads behind stores would wait for them
    u32x4_t low[FI][FJ / 2];
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      if (iw + x * 16 >= e.n) break;
#pragma unroll
      for (int y = 0; y < FJ; y += 2) low[x][y / 2] = load_raw(xl, (iw + x * 16 + c) * e.m + jw + y * 16 + of, 8);
    }
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      if (iw + x * 16 >= e.n) break;
      u32x4_t down[FJ / 2];
#pragma unroll
      for (int y = 0; y < FJ; y += 2) {
        float v[8], hi[8], lo[8];
        pair(x, y, v);
        const int64_t i = iw + x * 16 + c, j = jw + y * 16 + of;
        unpack8(lo, low[x][y / 2], false);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = t.a * lo[k] + v[k] * (1.0f / kA);
        if constexpr (FORM == kNext) {
          const u32x4_t h = pack8(v, false);
          unpack8(hi, h, false);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] -= hi[k];
          put(x, y * 2 + of / 8, h);
          down[y / 2] = pack8(v, false);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] *= 1.0f / kX;
          if (!tall) {
            const int left = e.cols - j < 8 ? (int)(e.cols - j) : 8;
            if (i < e.rows && left > 0) move8<P>(t, e, i * e.cols + j, left, v, copy_bf);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) turn[(y * 16 + of + k) * 17 + c] = v[k];
          }
        }
      }
      if constexpr (FORM == kNext) {
        flush(x, x_of(t, e, t.from ^ 1));
#pragma unroll
        for (int y = 0; y < FJ; y += 2) put(x, y * 2 + of / 8, down[y / 2]);
        flush(x, xl);
      }
      if constexpr (FORM == kLast) {
        if (tall) {
          // row j of the parameter, its elements i .. i + 7
#pragma unroll
          for (int h = 0; h < FJ / 2; ++h) {
            const int jr = h * 32 + (lane >> 1), part = (lane & 1) * 8;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = turn[jr * 17 + part + k];
            const int64_t j = jw + jr, i = iw + x * 16 + part;
            const int left = e.cols - i < 8 ? (int)(e.cols - i) : 8;
            if (j < e.rows && left > 0) move8<P>(t, e, j * e.cols + i, left, v, copy_bf);
          }
        }
      }
    }
  }
}

constexpr int kSizes[] = {256, 128, 64};  // of tiles

// Tiles of a product and the time of their rounds over the compute units, from the linear layer's stages (us): rounds of
// as many tiles as run at once, each of the longest depth's stages.
struct Cost {
  int per_cu;
  double alone, full, rest;
};
constexpr Cost kTileCosts[] = {{1, 1.45, 1.45, 8.5}, {2, 0.75, 1.02, 3.4}, {2, 0.33, 0.43, 3.0}};

int64_t tiles_of(const Entry& e, int form, int size) {
  const int64_t n = (e.n + size - 1) / size, m = (e.m + size - 1) / size;
  return form == kGram || form == kPolynomial ? n * (n + 1) / 2 : n * m;
}

int choose(const Table& t, int form) {
  const int64_t cus = layer_cus();
  int best = 0;
  double least = 0;
  for (int s = 0; s < 3; ++s) {
    int64_t tiles = 0;
    double work = 0, longest = 0;  // stages of all tiles, and of the deepest
    for (int i = 0; i < t.count; ++i) {
      const double depth = (form == kGram ? t.e[i].m : t.e[i].n) / BK;
      const int64_t k = tiles_of(t.e[i], form, kSizes[s]);
      tiles += k;
      work += (double)k * (depth * kTileCosts[s].full + kTileCosts[s].rest);
      const double one = depth * (tiles > cus ? kTileCosts[s].full : kTileCosts[s].alone) + kTileCosts[s].rest;
      longest = one > longest ? one : longest;
    }
    const int64_t slots = cus * kTileCosts[s].per_cu, rounds = (tiles + slots - 1) / slots;
    // whole rounds where the tiles are alike, the work shared evenly where there are many
    const double us = rounds <= 1 ? longest : 0.5 * (work / slots + longest) + 0.5 * rounds * (work / tiles);
    if (s == 0 || us < least) {
      least = us;
      best = s;
    }
  }
  return best;
}

template <int FORM, int P>
hipError_t run_form(Table t, int copy_bf, hipStream_t s) {
  const int size = choose(t, FORM);
  uint32_t total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = total;
    total += (uint32_t)tiles_of(t.e[i], FORM, kSizes[size]);
  }
  t.total = total;
  switch (size) {
    case 0: muon_kernel<FORM, P, 2, 4, 8, 4, 2><<<total, 512, 0, s>>>(t, copy_bf); break;
    case 1: muon_kernel<FORM, P, 2, 2, 4, 4, 2><<<total, 256, 0, s>>>(t, copy_bf); break;
    default: muon_kernel<FORM, P, 2, 2, 2, 2, 4><<<total, 256, 0, s>>>(t, copy_bf); break;
  }
  return hipGetLastError();
}

template <int G>
hipError_t run_start(Table t, hipStream_t s) {
  uint32_t total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = total;
    total += (uint32_t)(((int64_t)t.e[i].rows * t.e[i].cols + kChunk - 1) / kChunk);
  }
  muon_momentum_kernel<G><<<total, 256, 0, s>>>(t);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = total;
    total += (uint32_t)((int64_t)(t.e[i].n / 64) * (t.e[i].m / 64));
  }
  muon_start_kernel<G><<<total, 256, 0, s>>>(t);
  return hipGetLastError();
}

int64_t region(const Entry& e) {
  const int64_t chunks = ((int64_t)e.rows * e.cols + kChunk - 1) / kChunk;
  return (3 * x_bytes(e) + 2 * a_bytes(e) + chunks * 8 + 255) / 256 * 256;
}

Entry entry(const MuonMatrix& x) {
  Entry e = {};
  e.param = x.param;
  e.grad = x.grad;
  e.momentum = x.momentum;
  e.copy = x.copy;
  e.rows = (int32_t)x.rows;
  e.cols = (int32_t)x.cols;
  const int64_t n = x.rows < x.cols ? x.rows : x.cols, m = x.rows < x.cols ? x.cols : x.rows;
  e.n = (int32_t)((n + kPad - 1) / kPad * kPad);
  e.m = (int32_t)((m + kPad - 1) / kPad * kPad);
  return e;
}

// Matrices worked on together: until their X's tiles of 128 are this many, or the table is full. (25 matrices of
// 1024 x 4096 in groups of 1024 tiles 4.1 ms, of 2048 3.3, all at once 3.1: a launch of more tiles has less of a last
// round.)
constexpr int64_t kEnough = 16384;

// Calls f(first, end) for each group of matrices.
template <class F>
void groups(const MuonMatrix* x, int64_t count, F f) {
  int64_t from = 0, tiles = 0, in = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (x[i].rows == 0 || x[i].cols == 0) continue;
    tiles += tiles_of(entry(x[i]), kNext, 128);
    if (++in == kMost || tiles >= kEnough) {
      f(from, i + 1);
      from = i + 1;
      tiles = in = 0;
    }
  }
  if (in) f(from, count);
}

}  // namespace

size_t muon_workspace_bytes(const MuonMatrix* x, int64_t count) {
  int64_t most = 0;
  groups(x, count, [&](int64_t from, int64_t end) {
    int64_t n = 0;
    for (int64_t i = from; i < end; ++i)
      if (x[i].rows && x[i].cols) n += region(entry(x[i]));
    most = n > most ? n : most;
  });
  return (size_t)most;
}

hipError_t launch_muon(int pkind, int gkind, int ckind, const MuonMatrix* x, int64_t count, const MuonScalars& sc, void* ws,
                       hipStream_t s) {
  hipError_t e = hipSuccess;
  groups(x, count, [&](int64_t from, int64_t end) {
    if (e != hipSuccess) return;
    Table t = {};
    for (uint32_t& f : t.first) f = ~0u;
    t.ws = static_cast<char*>(ws);
    t.grad_scale = sc.grad_scale;
    t.mu = sc.mu;
    t.omu = sc.omu;
    t.eps = sc.eps;
    t.keep = sc.keep;
    t.a = sc.a;
    t.b = sc.b;
    t.c = sc.c;
    t.nesterov = sc.nesterov;
    t.apply = sc.apply;
    int64_t at = 0;
    for (int64_t i = from; i < end; ++i) {
      if (!x[i].rows || !x[i].cols) continue;
      Entry& o = t.e[t.count++];
      o = entry(x[i]);
      if (!sc.apply) {
        o.momentum = nullptr;
        o.copy = nullptr;
      }
      o.at = at;
      at += region(o);
      const double r = (double)x[i].rows, c = (double)x[i].cols;
      o.rate = (float)(sc.lr * (sc.by_rms ? 0.2 * sqrt(r > c ? r : c) : sqrt(r > c ? r / c : 1.0)));
    }
    e = gkind == FMX_DTYPE_F32 ? run_start<FMX_DTYPE_F32>(t, s) : gkind == FMX_DTYPE_BF16 ? run_start<FMX_DTYPE_BF16>(t, s)
                                                                                     : run_start<FMX_DTYPE_F16>(t, s);
    for (int k = 0; k < sc.steps && e == hipSuccess; ++k) {
      t.from = k & 1;
      e = run_form<kGram, 0>(t, 0, s);
      if (e == hipSuccess) e = run_form<kPolynomial, 0>(t, 0, s);
      if (e != hipSuccess) return;
      const int bf = ckind == FMX_DTYPE_BF16;
      if (k + 1 < sc.steps)
        e = run_form<kNext, 0>(t, 0, s);
      else if (pkind == FMX_DTYPE_F32)
        e = run_form<kLast, FMX_DTYPE_F32>(t, bf, s);
      else if (pkind == FMX_DTYPE_BF16)
        e = run_form<kLast, FMX_DTYPE_BF16>(t, bf, s);
      else
        e = run_form<kLast, FMX_DTYPE_F16>(t, bf, s);
    }
  });
  return e;
}

}  // namespace fmx
