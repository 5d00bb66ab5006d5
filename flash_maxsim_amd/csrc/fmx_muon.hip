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
//                            (thousands of matrices of 1 to 8 rows, whose few errors do not average out: median 1.5e-3 to
//                            2.6e-3, the largest 1.4e-2, of 2 x 2; of 16 rows and more 2.6e-3 at most)
// so X lies in memory as two fp16 arrays, of which the lower one is read and written by the epilogue alone (X = B X_upper +
// a X_lower): no product more. The last form saves the epilogue X's upper half (24 matrices of 1024 x 4096: 302 us a
// launch, 364 with it read; B's diagonal's rest as a product of its own in the loop 448). X is held times
// 2^8, A and B times 2^10: their small elements stay clear of fp16's subnormal ones.
//
// A and B are symmetric: tiles on and below the diagonal are computed, and a tile that lies below leaves LDS
// twice, the second time through transposing reads. Matrices taller than wide are transposed when X is made, and the
// last product's epilogue, which moves the parameters, transposes back.
//
// 25 matrices, 24 of 1024 x 4096, a step: 2.63 ms with bf16 parameters and gradients, 2.93 with float32 parameters, bf16
// gradients and copies, 2.98 with float32 gradients.
//
// A launch walks the tiles of up to kMost matrices of any shapes, from a table in its arguments: two for the momentum and X, three
// a step (A, B, X), two where the matrices are small.
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
constexpr int kChunk = 8192;                // elements whose squares one workgroup adds up, or a multiple (chunk_of)
// Sums of squares of a matrix at most: every workgroup that makes a tile of X adds all of them, 16 KB, four bytes an element of
// the tile. (Without a bound the work grows with the square of the elements: all before the first step 931 us for
// 8192 x 28672 bf16 and 268 ms for 4104 x 2^20; so 277 us and 7.2 ms.)
constexpr int kSums = 2048;

struct Entry {
  void* param;          // or the orthogonalised result
  const void* grad;
  float* momentum;      // or null: u is the gradient itself
  void* copy;
  int64_t at;           // of its part of the workspace, bytes
  int32_t rows, cols;   // of the parameter
  int32_t n, m;         // of X, padded: n the shorter side
  float rate;
  int32_t chunk;        // elements of a sum of squares
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
// waits for the arguments' memory once for every step (17 launches over four small matrices 102 -> 97 us).
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

// 8 float32 values past the caches, which are left to what is read again: the momentum is next read whole. (24 matrices of
// 1024 x 4096 224 -> 175 us for the launch; steps over 4 to 36 of them 1 to 3 % less, so too over 12 of 512 x 2048.)
__device__ __forceinline__ void store_past(float* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    typedef f32x4_t loose_t __attribute__((aligned(4)));
    __builtin_nontemporal_store(f32x4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<loose_t*>(p));
    __builtin_nontemporal_store(f32x4_t{v[4], v[5], v[6], v[7]}, reinterpret_cast<loose_t*>(p + 4));
  } else {
    store8<FMX_DTYPE_F32>(p, 0, left, v);
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
  for (int part = 0; part < e.chunk; part += kChunk) {
#pragma unroll
    for (int v = 0; v < kChunk / 2048; ++v) {
      const int64_t from = (int64_t)chunk * e.chunk + part + v * 2048 + threadIdx.x * 8;
      if (from >= size) break;
      const int left = size - from < 8 ? (int)(size - from) : 8;
      float g[8], m[8], u[8];
      load8<G>(g, e.grad, from, left);
      if (e.momentum) {
        load8<FMX_DTYPE_F32>(m, e.momentum, from, left);
#pragma unroll
        for (int k = 0; k < 8; ++k) m[k] = t.mu * m[k] + t.omu * (g[k] * scale);
        store_past(e.momentum + from, left, m);
      }
      direction(u, g, m, t, e.momentum != nullptr, scale);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += k < left ? (double)u[k] * (double)u[k] : 0.0;
    }
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
  const int64_t size = (int64_t)e.rows * e.cols, chunks = (size + e.chunk - 1) / e.chunk;
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
  // 8 lanes a row, a line of memory; rows r and r + 32 of the tile
  const int row = threadIdx.x >> 3, part = (threadIdx.x & 7) * 8;
  // the tile's rows as the parameter has them: of i, or of j
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  float x[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + row + 32 * h, c = c0 + part;
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
      for (int k = 0; k < 8; ++k) tile[part + k][row + 32 * h] = x[h][k];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 8; ++k) x[h][k] = tile[row + 32 * h][part + k];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t at = (int64_t)(i0 + row + 32 * h) * e.m + j0 + part;
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
    for (int k = 0; k < 8; ++k) x[k] = __builtin_fmaf(-e.rate, x[k], p[k] * t.keep);
  }
  store8<P>(e.param, at, left, x);
  if (P == FMX_DTYPE_F32 && e.copy) store16(e.copy, at, left, x, copy_bf);
}

// b A + c A^2 of an element, as B is held. (Multiplications and additions are fused as written here and in finish_x: a matrix
// has the same bits by whichever kernel.)
__device__ __forceinline__ float polynomial(const Table& t, float a, float square) {
  return __builtin_fmaf(t.b, a, t.c / kA * square);
}

// A lane's 8 neighbouring columns of a pair of j fragments; of a row-major operand the lanes exchange halves.
template <bool BMAJ>
__device__ __forceinline__ void pair_of(const f32x4_t& a, const f32x4_t& b, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = a[k];
    v[4 + k] = b[k];
    if constexpr (BMAJ) {
      const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v[k]),
                                                      __builtin_bit_cast(uint32_t, v[4 + k]), false, false);
      const uint32_t r0 = r[0], r1 = r[1];
      v[k] = __builtin_bit_cast(float, r0);
      v[4 + k] = __builtin_bit_cast(float, r1);
    }
  }
}

// From a wave's products of FI x FJ fragments, from row iw and column jw on, to the next X and its lower half (kNext) or to
// the parameter (kLast; P: its type), in whole lines: `mine` is LDS of the wave's own, kTurn bytes. What lies outside of X
// is left out.
constexpr int kTurn = 4096;
template <int FORM, int P, int FI, int FJ>
__device__ __forceinline__ void finish_x(const Table& t, const Entry& e, const f32x4_t (&acc)[FI][FJ], int64_t iw, int64_t jw,
                                         unsigned char* mine, int lane, int copy_bf) {
  constexpr int ROW = FJ * 32, CH = ROW / 16;  // bytes of a 16-bit row of the block, 16-byte pieces of it
  static_assert(16 * ROW <= kTurn && FJ * 16 * 16 * 4 <= kTurn, "a wave's block");
  const int c = lane & 15, g = lane >> 4, of = (g & 1) * 16 + (g >> 1) * 8;
  auto spot = [&](int r, int ch) __attribute__((always_inline)) { return mine + r * ROW + ((ch ^ (r & (CH - 1))) << 4); };
  auto put = [&](int ch, const u32x4_t& w) __attribute__((always_inline)) { *reinterpret_cast<u32x4_t*>(spot(c, ch)) = w; };
  // the block's first element: its others lie within 128 rows of at most 2^21 bytes, below 2^31
  const int64_t first = iw * e.m + jw;
  const int pitch = e.m * 2, rows = jw < e.m ? (int)(e.n - iw) : 0;
  const uint32_t out_at = (uint32_t)((lane / CH) * pitch + (lane % CH) * 16), in_at = (uint32_t)(c * pitch + of * 2);
  auto flush = [&](int x, rsrc_t out) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 16 * CH / 64; ++h) {
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(spot(h * (64 / CH) + lane / CH, lane % CH));
      __builtin_amdgcn_raw_buffer_store_b128(w, out, x * 16 < rows ? out_at : kOOB, (x * 16 + h * (64 / CH)) * pitch, 0);
    }
  };
  const rsrc_t rl = make_rsrc(low_of(t, e) + first, 0x7fffffffu);
  const rsrc_t rx = make_rsrc(x_of(t, e, t.from ^ 1) + first, 0x7fffffffu);
  const bool tall = e.rows > e.cols;
  // kLast of a tall parameter: [FJ * 16][16], a 16-row block turned round, its columns swizzled
  float* turn = reinterpret_cast<float*>(mine);
  auto turned = [&](int j, int i) __attribute__((always_inline)) { return j * 16 + (i ^ (j & 15)); };
  // Everything that is read, before the first store: loads behind stores would wait for them. (No branches: rows past X's
  // read as zeros, and what is stored to them goes nowhere.)
  u32x4_t low[FI][FJ / 2];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; y += 2)
      low[x][y / 2] = __builtin_amdgcn_raw_buffer_load_b128(rl, x * 16 < rows ? in_at + y * 32 : kOOB, x * 16 * pitch, 0);
#pragma unroll
  for (int x = 0; x < FI; ++x) {
    u32x4_t down[FJ / 2];
#pragma unroll
    for (int y = 0; y < FJ; y += 2) {
      float v[8], hi[8], lo[8];
      pair_of<true>(acc[x][y], acc[x][y + 1], v);
      const int64_t i = iw + x * 16 + c, j = jw + y * 16 + of;
      unpack8(lo, low[x][y / 2], false);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __builtin_fmaf(t.a, lo[k], v[k] * (1.0f / kA));
      if constexpr (FORM == kNext) {
        const u32x4_t h = pack8(v, false);
        unpack8(hi, h, false);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] -= hi[k];
        put(y * 2 + of / 8, h);
        down[y / 2] = pack8(v, false);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= 1.0f / kX;
        if (!tall) {
          const int left = e.cols - j < 8 ? (int)(e.cols - j) : 8;
          if (i < e.rows && left > 0) move8<P>(t, e, i * e.cols + j, left, v, copy_bf);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) turn[turned(y * 16 + of + k, c)] = v[k];
        }
      }
    }
    if constexpr (FORM == kNext) {
      flush(x, rx);
#pragma unroll
      for (int y = 0; y < FJ; y += 2) put(y * 2 + of / 8, down[y / 2]);
      flush(x, rl);
    }
    if constexpr (FORM == kLast) {
      if (tall) {
        // row j of the parameter, its elements i .. i + 7
#pragma unroll
        for (int h = 0; h < FJ / 2; ++h) {
          const int jr = h * 32 + (lane >> 1), part = (lane & 1) * 8;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = turn[turned(jr, part + k)];
          const int64_t j = jw + jr, i = iw + x * 16 + part;
          const int left = e.cols - i < 8 ? (int)(e.cols - i) : 8;
          if (j < e.rows && left > 0) move8<P>(t, e, j * e.cols + i, left, v, copy_bf);
        }
      }
    }
  }
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
  const int c = lane & 15, g = lane >> 4, of = 8 * g;
  stage_barrier();  // LDS is free: nothing is loaded into it or read from it any more
  constexpr int ROW = FJ * 32;  // bytes of a wave's 16-bit row
  unsigned char* mine = (wave < WI * WJ / 2 ? lds0 : lds1) + (wave % (WI * WJ / 2)) * (BYTES / (WI * WJ / 2));
  static_assert(BYTES / (WI * WJ / 2) >= FI * 16 * ROW && BYTES / (WI * WJ / 2) >= kTurn, "a wave's block");
  const int64_t iw = i0 + wi * FI * 16, jw = j0 + wj * FJ * 16;
  if (jw >= width || iw >= e.n) return;  // sides are multiples of 64 and a wave's block begins at one of 32 at least

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
        pair_of<false>(acc[x][y], acc[x][y + 1], v);
        const int64_t at = (iw + x * 16 + c) * e.n + jw + y * 16 + of;
        if constexpr (FORM == kGram) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] *= kA / (kX * kX);
        } else {
          float w[8];
          load16(w, in, at, 8, false);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = polynomial(t, w[k], v[k]);
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
    finish_x<FORM, P, FI, FJ>(t, e, acc, iw, jw, mine, lane, copy_bf);
  }
}

// X's products in tiles of 256 x 256: a workgroup on each compute unit takes tile after tile, the next one's first two stages
// are loaded before a tile is finished, and its stores drain while the next tile's first stage is multiplied. (24 matrices of
// 1024 x 4096 311 -> 294 us. The products alone take 206 of them, what is read and written besides 150: they share the unit's
// path to the caches, and of the 990 MB that HBM moves 400 are stores. Not waiting for those in the first stage took
// registers that spilled, 305; starting the units at different times and storing past the caches gained nothing.)
template <int FORM, int P>
__global__ void __launch_bounds__(512) muon_next_kernel(Table t, int copy_bf) {
  constexpr int WI = 2, FI = 8, FJ = 4, TI = 256, NT = 512, BYTES = 2 * TI * BK * 2;
  using SideA = Side<false, false, TI, NT>;
  using SideB = Side<true, false, TI, NT>;
  constexpr int LOADS = SideA::kLoads + SideB::kLoads, READS = 2 * FJ + FI;
  __shared__ __attribute__((aligned(1024))) unsigned char lds0[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds1[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char own[8 * kTurn];

  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave % WI, wj = wave / WI;
  Frags<false, false, TI> fa(wi * FI * 16, tid & 63);
  Frags<true, false, TI> fb(wj * FJ * 16, tid & 63);
  // Addresses made of these are made anew for every tile, and hold no registers where they are not used.
  auto fresh = [](auto& v) __attribute__((always_inline)) { __asm__ volatile("" : "+v"(v)); };
  struct Tile {
    int at, i0;
    int64_t j0;
  };
  auto place = [&](uint32_t id) __attribute__((always_inline)) {
    // workgroups go to the eight XCDs in turn; each XCD takes a run of consecutive tiles
    const uint32_t per = t.total / 8, x = id & 7, rest = t.total & 7;
    return (id >> 3) + x * per + (x < rest ? x : rest);
  };
  auto locate = [&](uint32_t id, int at) __attribute__((always_inline)) {
    Tile o;
    o.at = at;
    const Entry& e = t.e[o.at];
    id -= t.first[o.at];
    // the rows of a column of tiles, which read the same columns of X, one after the other
    const uint32_t ti = (uint32_t)(e.n + TI - 1) / TI, col = id / ti;
    o.i0 = (int)(id - col * ti) * TI;
    o.j0 = (int64_t)col * TI;
    return o;
  };
  // What a tile's stages are loaded from, as Side loads them, with what all lanes share in scalar registers: a thread's
  // chunks of B lie 64 rows apart, those of X 16, and sides are multiples of 64.
  const char *pa, *pb;
  int depth, rows, pitch;
  uint32_t va_at, vb_at;
  auto begin = [&](const Tile& o) __attribute__((always_inline)) {
    const Entry& e = t.e[o.at];
    pa = reinterpret_cast<const char*>(b_of(t, e) + (int64_t)o.i0 * e.n);
    pb = reinterpret_cast<const char*>(x_of(t, e, t.from) + o.j0);
    depth = e.n;
    rows = e.n - o.i0;
    pitch = e.m * 2;
    const int ra = tid / 8, rb = tid / 32;
    const int ca = (tid % 8) ^ SideA::key(ra), cb = (tid % 32) ^ SideB::key(rb);
    va_at = (uint32_t)(ra * depth * 2 + ca * 16);
    vb_at = o.j0 + cb * 8 < e.m ? (uint32_t)(rb * pitch + cb * 16) : kOOB;
  };
  const uint32_t first = place(blockIdx.x);
  Tile o = locate(first, __builtin_amdgcn_readfirstlane(entry_of(t, first)));
  begin(o);
  f32x4_t acc[FI][FJ];
  u32x4_t va[2][FI], vb[2][FJ];
  // stage `it`; past the last one zeros
  auto issue = [&](unsigned char* lds, int it) __attribute__((always_inline)) {
    const bool have = it * BK < depth;
    const char *a = pa + it * BK * 2, *b = pb + (int64_t)it * BK * pitch;
#pragma unroll
    for (int n = 0; n < SideA::kLoads; ++n)
      dma16_lds<false>(make_rsrc(a + (int64_t)(n * 64) * depth * 2, 0x7fffffffu), lds + (n * NT + wave * 64) * 16,
                       have && n * 64 < rows ? va_at : kOOB);
#pragma unroll
    for (int n = 0; n < SideB::kLoads; ++n)
      dma16_lds<false>(make_rsrc(b + (int64_t)(n * 16) * pitch, 0x7fffffffu), lds + TI * BK * 2 + (n * NT + wave * 64) * 16,
                       have ? vb_at : kOOB);
  };
  auto read = [&](auto set, const unsigned char* lds, int kk) __attribute__((always_inline)) {
    constexpr int Z = decltype(set)::value;
#pragma unroll
    for (int y = 0; y < FJ; ++y) vb[Z][y] = fb.read(lds + TI * BK * 2, y, kk);
    fresh(fa.at[kk]);
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
  // The stage in `lds`, while stage `it` (of this tile or the next) is loaded behind it and, unless it is the tile's last,
  // the first fragments of the one in `other` are read: run_stages' order.
  auto stage = [&](unsigned char* lds, const unsigned char* other, int it, auto last) __attribute__((always_inline)) {
    read(set1, lds, 1);
    multiply(set0);
    wait_vmem<0>();
    stage_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue(lds, it);
    if constexpr (!decltype(last)::value) read(set0, other, 0);
    multiply(set1);
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    if constexpr (!decltype(last)::value) {
#pragma unroll
      for (int n = 0; n < READS / 2; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x008, FI * FJ, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::false_type more_follow{};
  constexpr std::true_type last_one{};
  issue(lds0, 0);
  issue(lds1, 1);
  wait_vmem<LOADS>();
  stage_barrier();
  for (uint32_t id = blockIdx.x;; id += gridDim.x) {
    fresh(fb.at[0]);
    read(set0, lds0, 0);
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int nit = (depth + 2 * BK - 1) / (2 * BK) * 2;  // in pairs: a tile begins in lds0 (a stage past the end is zeros)
    for (int it = 2; it < nit; it += 2) {
      stage(lds0, lds1, it, more_follow);
      stage(lds1, lds0, it + 1, more_follow);
    }
    const Tile now = o;
    const bool more = id + gridDim.x < t.total;
    fresh(tid);
    if (more) {
      // from the last tile's entry on, by scalar loads: entry_of's would wait for the stages in flight
      const uint32_t next = place(id + gridDim.x);
      int at = o.at;
      while (at + 1 < t.count && t.first[at + 1] <= next) ++at;
      while (t.first[at] > next) --at;
      o = locate(next, at);
      begin(o);
    } else {
      depth = 0;  // nothing is read, zeros reach LDS
    }
    stage(lds0, lds1, 0, more_follow);
    stage(lds1, lds0, 1, last_one);
    const Entry& e = t.e[now.at];
    const int64_t jw = now.j0 + wj * FJ * 16;
    fresh(tid);
    finish_x<FORM, P, FI, FJ>(t, e, acc, now.i0 + wi * FI * 16, jw, own + wave * kTurn, tid & 63, copy_bf);
    if (!more) break;
  }
  wait_vmem<0>();  // the empty stages' DMA writes no longer reach LDS after this wave ends
}

// Small matrices (n up to kSmall, all tiles of a launch at once): a product's launch for X makes its rows of B itself, from
// all of A in LDS, and B has no launch of its own: 64 x 64 of X a workgroup, 64 x n of B before. (Five steps over matrices of,
// us: 64 x 1024 82 -> 67, 128 x 768 83 -> 66, 256 x 256 80 -> 69, four of 256 x 1024 101 -> 92; launch by launch of those 4.7 and
// 5.4 -> 8.1. Eight stages in LDS for their Gram matrices: 256 x 4096 159 -> 148, 256 x 1024 the same, 256 x 256 69 -> 71: not kept.)
constexpr int kSmall = 256;
template <int FORM, int P>
__global__ void __launch_bounds__(256) muon_small_kernel(Table t, int copy_bf) {
  constexpr int FI = 2, FJ = 2, BLOCK = 64 * BK * 2, NB = kSmall / 64;  // 64 x 64 elements of 16 bits
  using SideA = Side<false, false, 64, 256>;
  using SideX = Side<true, false, 64, 256>;
  __shared__ __attribute__((aligned(1024))) unsigned char all[NB * NB * BLOCK];  // A by blocks, then X's columns
  __shared__ __attribute__((aligned(1024))) unsigned char panel[NB * BLOCK];     // B's rows
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave & 1, wj = wave >> 1;
  // workgroups go to the eight XCDs in turn; each XCD takes a run of consecutive tiles
  uint32_t id = blockIdx.x;
  {
    const uint32_t per = t.total / 8, x = id & 7, rest = t.total & 7;
    id = (id >> 3) + x * per + (x < rest ? x : rest);
  }
  const int at = __builtin_amdgcn_readfirstlane(entry_of(t, id));
  const Entry& e = t.e[at];
  id -= t.first[at];
  const int nb = e.n / 64;
  const int col = (int)id / nb, row = (int)id - col * nb;
  const int64_t j0 = (int64_t)col * 64;

  const int r = tid >> 3, ch = tid & 7;  // a thread's 16 bytes of 32 rows of 128
  const rsrc_t ra = make_rsrc(a_of(t, e), 0x7fffffffu);
  for (int b = 0; b < nb; ++b)
    for (int k = 0; k < nb; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        dma16_lds<false>(ra, all + (b * nb + k) * BLOCK + (h * 256 + wave * 64) * 16,
                         (uint32_t)(((b * 64 + h * 32 + r) * e.n + k * 64 + (ch ^ SideA::key(r)) * 8) * 2));
  // X's columns wait in registers until A's place is free
  const rsrc_t rx = make_rsrc(x_of(t, e, t.from) + j0, 0x7fffffffu);
  u32x4_t x[2 * NB];
#pragma unroll
  for (int q = 0; q < 2 * NB; ++q)
    x[q] = ld16(rx, q * 32 < e.n ? (uint32_t)(((q * 32 + r) * (int64_t)e.m + ch * 8) * 2) : kOOB);
  wait_vmem<0>();
  stage_barrier();

  const Frags<false, false, 64> fi(wi * 32, lane), fj(wj * 32, lane);
  // of row i of a block of B and columns j .. j + 3 of it: where they lie in A's and the panel's blocks
  auto spot = [&](int i, int j) __attribute__((always_inline)) { return i * 128 + (((j >> 3) ^ (i & 7)) << 4) + (j & 4) * 2; };
  f32x4_t acc[FI][FJ];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
      for (int b = 0; b < FJ; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  auto multiply = [&](const u32x4_t (&vi)[FI], const u32x4_t (&vj)[FJ]) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
      for (int b = 0; b < FJ; ++b) acc[a][b] = mfma16x16x32<false>(vj[b], vi[a], acc[a][b]);
  };
  // Both products for a count of blocks that the compiler knows: fragments are then read well ahead of their multiplication,
  // and those of the panel's own rows once.
  auto products = [&](auto blocks) __attribute__((always_inline)) {
    constexpr int N = decltype(blocks)::value;
    u32x4_t vi[2 * N][FI];
#pragma unroll
    for (int k = 0; k < 2 * N; ++k)
#pragma unroll
      for (int a = 0; a < FI; ++a) vi[k][a] = fi.read(all + (row * N + k / 2) * BLOCK, a, k & 1);
#pragma unroll 1
    for (int jb = 0; jb < N; ++jb) {
      clear();
#pragma unroll
      for (int k = 0; k < 2 * N; ++k) {
        const unsigned char* aj = all + (jb * N + k / 2) * BLOCK;
        const u32x4_t vj[FJ] = {fj.read(aj, 0, k & 1), fj.read(aj, 1, k & 1)};
        multiply(vi[k], vj);
      }
#pragma unroll
      for (int a = 0; a < FI; ++a)
#pragma unroll
        for (int b = 0; b < FJ; ++b) {
          const int i = wi * 32 + a * 16 + c, j = wj * 32 + b * 16 + 4 * g;
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(all + (row * N + jb) * BLOCK + spot(i, j));
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = polynomial(t, unpack((k & 1) ? w[k / 2] >> 16 : w[k / 2] & 0xffffu, false), acc[a][b][k]);
            v[k] += row == jb && i == j + k ? t.a * kA : 0.0f;
          }
          *reinterpret_cast<u32x2_t*>(panel + jb * BLOCK + spot(i, j)) =
              u32x2_t{pack2(v[0], v[1], false), pack2(v[2], v[3], false)};
        }
    }
    stage_barrier();  // A is not read any more
#pragma unroll
    for (int q = 0; q < 2 * N; ++q)
      *reinterpret_cast<u32x4_t*>(all + (q * 32 + r) * 128 + ((ch ^ SideX::key(r)) << 4)) = x[q];
    stage_barrier();
    const Frags<true, false, 64> fx(wj * 32, lane);
    clear();
#pragma unroll
    for (int k = 0; k < 2 * N; ++k) {
      const unsigned char *bi = panel + (k / 2) * BLOCK, *xj = all + (k / 2) * BLOCK;
      const u32x4_t vb[FI] = {fi.read(bi, 0, k & 1), fi.read(bi, 1, k & 1)}, vx[FJ] = {fx.read(xj, 0, k & 1), fx.read(xj, 1, k & 1)};
      multiply(vb, vx);
    }
  };
  switch (nb) {
    case 1: products(std::integral_constant<int, 1>{}); break;
    case 2: products(std::integral_constant<int, 2>{}); break;
    case 3: products(std::integral_constant<int, 3>{}); break;
    default: products(std::integral_constant<int, NB>{}); break;
  }
  // past X's columns there is room in A's place
  static_assert(NB * BLOCK + 4 * kTurn <= NB * NB * BLOCK, "LDS of the waves' own");
  finish_x<FORM, P, FI, FJ>(t, e, acc, row * 64 + wi * 32, j0 + wj * 32, all + NB * BLOCK + wave * kTurn, lane, copy_bf);
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
    case 0:
      if constexpr (FORM == kGram || FORM == kPolynomial) {
        muon_kernel<FORM, P, 2, 4, 8, 4, 2><<<total, 512, 0, s>>>(t, copy_bf);
      } else {
        const uint32_t cus = (uint32_t)layer_cus();
        muon_next_kernel<FORM, P><<<total < cus ? total : cus, 512, 0, s>>>(t, copy_bf);
      }
      break;
    case 1: muon_kernel<FORM, P, 2, 2, 4, 4, 2><<<total, 256, 0, s>>>(t, copy_bf); break;
    default: muon_kernel<FORM, P, 2, 2, 2, 2, 4><<<total, 256, 0, s>>>(t, copy_bf); break;
  }
  return hipGetLastError();
}

// Whether muon_small_kernel takes a launch's matrices.
bool small(const Table& t) {
  int64_t tiles = 0;
  for (int i = 0; i < t.count; ++i) {
    if (t.e[i].n > kSmall) return false;
    tiles += tiles_of(t.e[i], kNext, 64);
  }
  return tiles <= layer_cus();
}

template <int FORM, int P>
hipError_t run_small(Table t, int copy_bf, hipStream_t s) {
  t.total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = t.total;
    t.total += (uint32_t)tiles_of(t.e[i], FORM, 64);
  }
  muon_small_kernel<FORM, P><<<t.total, 256, 0, s>>>(t, copy_bf);
  return hipGetLastError();
}

// The next X, or (kLast) the parameters.
template <int FORM, int P>
hipError_t run_x(const Table& t, bool few, int copy_bf, hipStream_t s) {
  return few ? run_small<FORM, P>(t, copy_bf, s) : run_form<FORM, P>(t, copy_bf, s);
}

// Elements of a matrix's sum of squares: kChunk, or as many times that as keep to kSums sums.
int32_t chunk_of(int64_t size) { return (int32_t)((size + (int64_t)kChunk * kSums - 1) / ((int64_t)kChunk * kSums) * kChunk); }
int64_t chunks_of(const Entry& e) { return ((int64_t)e.rows * e.cols + e.chunk - 1) / e.chunk; }

template <int G>
hipError_t run_start(Table t, hipStream_t s) {
  uint32_t total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = total;
    total += (uint32_t)chunks_of(t.e[i]);
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
  return (3 * x_bytes(e) + 2 * a_bytes(e) + chunks_of(e) * 8 + 255) / 256 * 256;
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
  e.chunk = chunk_of(x.rows * x.cols);
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
    const bool few = small(t);
    for (int k = 0; k < sc.steps && e == hipSuccess; ++k) {
      t.from = k & 1;
      e = run_form<kGram, 0>(t, 0, s);
      if (e == hipSuccess && !few) e = run_form<kPolynomial, 0>(t, 0, s);
      if (e != hipSuccess) return;
      const int bf = ckind == FMX_DTYPE_BF16;
      if (k + 1 < sc.steps)
        e = run_x<kNext, 0>(t, few, 0, s);
      else if (pkind == FMX_DTYPE_F32)
        e = run_x<kLast, FMX_DTYPE_F32>(t, few, bf, s);
      else if (pkind == FMX_DTYPE_BF16)
        e = run_x<kLast, FMX_DTYPE_BF16>(t, few, bf, s);
      else
        e = run_x<kLast, FMX_DTYPE_F16>(t, few, bf, s);
    }
  });
  return e;
}

}  // namespace fmx
