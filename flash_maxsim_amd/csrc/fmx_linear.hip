// Linear layer on MFMA: y = act(x W^T + b) + r, and the products of its backward.
//
// One kernel computes C[i, j] = sum_k A(i, k) B(j, k) for all three:
//   forward  i = row,  j = output,  k = input:  A = x [i, k],   B = W [j, k]
//   dx       i = row,  j = input,   k = output: A = dz [i, k],  B = W [k, j]
//   dw       i = out,  j = input,   k = row:    A = dz [k, i],  B = x [k, j]
// An operand stored [i, k] ("K-major") is read from LDS with 16-byte reads of 8
// k values; one stored [k, i] ("row-major") with transposing reads
// (ds_read_b64_tr_b16: of the 16 lanes that read a 4 x 16 block, lane l gets
// column l), so no operand is transposed in memory first.
//
// A workgroup computes a TI x TJ tile, its waves TI / WI x TJ / WJ each in
// registers. Stages of BK k values stream global -> LDS by DMA (16 bytes a
// lane) into NS buffers, the next stage in flight while one is multiplied.
// Chunk positions in LDS are XOR-swizzled so that the lanes of a read fall in
// distinct banks. C's j runs along the MFMA's result rows, so a lane holds 4
// (K-major B: 8, W's rows being read in a permuted order) consecutive outputs
// of one row and stores them together.
//
// A product whose tiles do not fill the GPU, or whose k is much longer than
// its tiles are many, is split over k: float32 partial tiles go to the
// workspace and a second kernel adds them in order (no atomics) and applies
// the epilogue.
#include "fmx_device.h"
#include "fmx_layers.h"
#include "fmx_product.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

// Slopes lie within -0.13 .. 1.13 and go from the forward to the backward in 16 bits, which get finer towards zero:
// GELU's slope at -5 is -7e-6, and a unit whose arguments all lie there learns by it (steps of 2^-14 made it zero). The
// bits of |slope| as float32, a measure of its logarithm, are shifted right by S, which divides the exponent by 2^S: a
// root drawn with straight lines from power to power of two. The code is that root in steps of 1 / 32767; it is kOne
// for a slope of 1, and the largest slope is below 32766. What a slope is off by, half a step, is
//   fp16, S = 1  2^-15 for 1/2 to 1 (twice that above), at most 2^-14 of it down to 0.28, twice that for each
//                two powers of two further down; 2^-30 is the smallest that is not zero (fp16's own: 2^-24)
//   bf16, S = 2  2^-14 for 1/2 to 1, at most 2^-13 of it down to 0.07, twice that for each four powers of two;
//                2^-60, where squares of gradients leave float32
// 0 and 1 are exact. Beside dz's rounding to the operands' type (2^-11, 2^-8) that adds a hundredth to the gradients'
// error; rounding z itself made them up to 1.57 times as far from 64 bits as ones rounded once (1.41 is what the
// rounding of dz and of the result make). The backward needs no exponentials. NaN's bits give the code 32767 at
// either sign.
template <bool BF>
struct SlopeCode {
  static constexpr int S = BF ? 2 : 1;
  static constexpr float kStep = 1.0f / 32767.0f, kOne = BF ? 32230.0f : 31700.0f;
  static constexpr uint32_t kBias = __builtin_bit_cast(uint32_t, kOne * kStep) - (0x3f800000u >> S);
};
template <bool BF>
__device__ __forceinline__ float slope_root(float a) {
  const uint32_t u = __builtin_bit_cast(uint32_t, a) & 0x7fffffffu;
  return __builtin_copysignf(__builtin_bit_cast(float, (u >> SlopeCode<BF>::S) + SlopeCode<BF>::kBias), a);
}
template <bool BF>
__device__ __forceinline__ uint32_t slopes2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_i16(slope_root<BF>(a), slope_root<BF>(b)));
}
template <bool BF>
__device__ __forceinline__ float slope_of(uint32_t bits16) {
  using C = SlopeCode<BF>;
  const float root = (float)(int16_t)bits16 * C::kStep;
  const uint32_t u = __builtin_bit_cast(uint32_t, root) & 0x7fffffffu;
  const float v = __builtin_bit_cast(float, ((u > C::kBias ? u : C::kBias) - C::kBias) << C::S);
  return u < 0x3f800000u ? __builtin_copysignf(v, root) : __builtin_nanf("");
}

template <bool BF>
__device__ __forceinline__ u32x4_t slopes8(const float (&s)[8]) {
  return u32x4_t{slopes2<BF>(s[0], s[1]), slopes2<BF>(s[2], s[3]), slopes2<BF>(s[4], s[5]), slopes2<BF>(s[6], s[7])};
}

// Products in v (the bias added already) to their place: the activation, its slope, the residual in `res`, y.
template <bool BF, int EPI>
__device__ __forceinline__ void finish(const LinearArgs& a, void* out, int64_t i, int64_t j, int left, float (&v)[8],
                                       const u32x4_t& res) {
  if constexpr (EPI != kNoEpilogue) {
    if constexpr (EPI != FMX_ACT_NONE) {
      float s[8];
      if (a.slope) {
        activate<EPI, true>(v, s, a.act);
        store_raw(a.slope, i * a.J + j, left, slopes8<BF>(s));
      } else {
        activate<EPI, false>(v, s, a.act);
      }
    }
    if (a.res) {
      float r[8];
      unpack8(r, res, BF);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += r[k];
    }
  }
  store16(out, i * a.J + j, left, v, BF);
}

// ---- the product ----

// PAIRED (a gated layer's backward): in dx k runs over the rows of B and then over those of B2, which A's columns meet
// after `half` stages; dw makes y from A and y2 from A2, whose tiles follow each other.
template <bool BF, bool AMAJ, bool BMAJ, int WI, int WJ, int FI, int FJ, int NS, int EPI, bool PAIRED>
__global__ void __launch_bounds__(WI* WJ * 64) linear_kernel(LinearArgs a) {
  constexpr int TI = WI * FI * 16, TJ = WJ * FJ * 16, NT = WI * WJ * 64;
  constexpr int BYTES = (TI + TJ) * BK * 2;
  using SideA = Side<AMAJ, false, TI, NT>;
  using SideB = Side<BMAJ, !BMAJ, TJ, NT>;
  constexpr int LOADS = SideA::kLoads + SideB::kLoads;
  __shared__ __attribute__((aligned(1024))) unsigned char lds0[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds1[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds2[NS > 2 ? BYTES : 16];
  __shared__ __attribute__((aligned(1024))) unsigned char lds3[NS > 2 ? BYTES : 16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave % WI, wj = wave / WI;

  const Place at(blockIdx.x, (uint32_t)a.ti, (uint32_t)a.tj, (uint32_t)a.splits, (uint32_t)a.band);
  const uint32_t split = at.split;
  const bool second = PAIRED && AMAJ && at.row >= (uint32_t)a.half;
  const int64_t i0 = (int64_t)(second ? at.row - (uint32_t)a.half : at.row) * TI, j0 = (int64_t)at.col * TJ;
  void* const out = second ? a.y2 : a.y;
  const int64_t k0 = (int64_t)split * a.split_k;
  const int64_t kn = a.K - k0 < a.split_k ? a.K - k0 : a.split_k;
  const int nit = (int)((kn + BK - 1) / BK);

  constexpr bool TURNS = PAIRED && !AMAJ;
  const SideA sa(second ? a.A2 : a.A, a.sa, i0, a.I, k0, tid);
  const SideB sb(a.B, a.sb, j0, a.Jr, TURNS ? 0 : k0, tid);
  const SideB sb2(TURNS ? a.B2 : a.B, TURNS ? a.sb2 : a.sb, j0, a.Jr, TURNS ? 0 : k0, tid);
  const Frags<AMAJ, false, TI> fa(wi * FI * 16, lane);
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
    const int left = (int)kn - it * BK;
    sa.issue(lds, it, left, wave);
    if constexpr (TURNS) {
      const int stage = (int)(k0 / BK) + it, own = stage < a.half ? stage : stage - a.half;
      if (stage < a.half)
        sb.issue(lds + TI * BK * 2, own, a.kb - own * BK, wave);
      else
        sb2.issue(lds + TI * BK * 2, own, a.kb - own * BK, wave);
    } else {
      sb.issue(lds + TI * BK * 2, it, left, wave);
    }
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
      for (int y = 0; y < FJ; ++y) acc[x][y] = mfma16x16x32<BF>(vb[Z][y], va[Z][x], acc[x][y]);
  };
  // dw: the sums of A's columns (db), by a product with ones in the waves that hold the tile's first columns of C
  constexpr bool SUMS = AMAJ && BMAJ && FI <= 4;
  const bool sums = SUMS && a.db_beside && j0 == 0 && wj == 0;
  f32x4_t total[SUMS ? FI : 1];
#pragma unroll
  for (int x = 0; x < (SUMS ? FI : 1); ++x) total[x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto add_up = [&](auto set) __attribute__((always_inline)) {
    if constexpr (SUMS) {
      const uint32_t one = BF ? 0x3f803f80u : 0x3c003c00u;
      if (sums) {
#pragma unroll
        for (int x = 0; x < FI; ++x)
          total[x] = mfma16x16x32<BF>(u32x4_t{one, one, one, one}, va[decltype(set)::value][x], total[x]);
      }
    }
  };
  run_stages<NS, LOADS, FJ*(BMAJ ? 2 : 1) + FI*(AMAJ ? 2 : 1), FI * FJ>(nit, buffer, issue, read, multiply, add_up);

  if constexpr (SUMS) {
    if (sums && lane < 16) {  // every row of the product with ones is the sums
#pragma unroll
      for (int x = 0; x < FI; ++x) {
        const int64_t i = i0 + wi * FI * 16 + x * 16 + lane;
        if (i < a.I) a.db_part[(int64_t)split * a.I + i] = total[x][0];
      }
    }
  }

  // A lane's results: row c of each i fragment, and of a pair of j fragments 8 columns. K-major B: its rows
  // were read so that they are consecutive. Row-major B: fragments y and y + 1 hold columns 4 g .. + 3 each, of
  // which an exchange between neighbouring 16-lane groups makes 8 of y (even g) or of y + 1 (odd g).
  const int c = lane & 15, g = lane >> 4;
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
  if (FJ == 4 && a.splits == 1 && i0 + TI <= a.I && j0 + TJ <= a.J) {
    // A whole tile: a wave turns its 16 x 64 blocks into rows of 128 bytes, whole lines of memory, in LDS
    // that nothing is read from or loaded into any more.
    wait_vmem<0>();
    stage_barrier();
    unsigned char* mine = (wave < WI * WJ / 2 ? lds0 : lds1) + (wave % (WI * WJ / 2)) * (BYTES / (WI * WJ / 2));
    const int64_t jw = j0 + wj * FJ * 16;
    float b[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 8; ++k) b[h][k] = 0.0f;
      if (EPI != kNoEpilogue && a.bias) load16(b[h], a.bias, jw + 32 * h + (BMAJ ? (g & 1) * 16 + (g >> 1) * 8 : 8 * g), 8, BF);
    }
    const int row = lane >> 3, ch = lane & 7;
    auto put = [&](int x, int h, const u32x4_t& w) __attribute__((always_inline)) {
      const int at = 4 * h + (BMAJ ? (g & 1) * 2 + (g >> 1) : g);
      *reinterpret_cast<u32x4_t*>(mine + x * 2048 + c * 128 + ((at ^ (c & 7)) << 4)) = w;
    };
    auto flush = [&](int x, void* out) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + x * 2048 + (row + 8 * h) * 128 + ((ch ^ row) << 4));
        const int64_t i = i0 + wi * FI * 16 + x * 16 + row + 8 * h;
        store_raw(out, i * a.J + jw + ch * 8, 8, w);
      }
    };
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      float v[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pair(x, 2 * h, v[h]);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[h][k] += b[h][k];
      }
      if constexpr (EPI != kNoEpilogue) {
        if constexpr (EPI != FMX_ACT_NONE) {
          float s[8];
          if (a.slope) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              activate<EPI, true>(v[h], s, a.act);
              put(x, h, slopes8<BF>(s));
            }
            flush(x, a.slope);
          } else {
            activate<EPI, false>(v[0], s, a.act);
            activate<EPI, false>(v[1], s, a.act);
          }
        }
        if (a.res) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t i = i0 + wi * FI * 16 + x * 16 + c, j = jw + 32 * h + 8 * g;
            float r[8];
            load16(r, a.res, i * a.sres + j, 8, BF);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[h][k] += r[k];
          }
        }
      }
      put(x, 0, pack8(v[0], BF));
      put(x, 1, pack8(v[1], BF));
      flush(x, out);
    }
    return;
  }
#pragma unroll
  for (int y = 0; y < FJ; y += 2) {
    const int64_t j = j0 + wj * FJ * 16 + y * 16 + (BMAJ ? (g & 1) * 16 + (g >> 1) * 8 : 8 * g);
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);  // columns inside; none: nothing is stored
    float b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = 0.0f;
    if (EPI != kNoEpilogue && a.bias && a.splits == 1 && left > 0) load16(b, a.bias, j, left, BF);
    // all of the residual before the first store: loads behind stores would wait for them
    u32x4_t res[FI];
    if (EPI != kNoEpilogue && a.res && a.splits == 1) {
#pragma unroll
      for (int x = 0; x < FI; ++x) {
        const int64_t i = i0 + wi * FI * 16 + x * 16 + c;
        res[x] = i < a.I && left > 0 ? load_raw(a.res, i * a.sres + j, left) : u32x4_t{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      const int64_t i = i0 + wi * FI * 16 + x * 16 + c;
      float v[8];
      pair(x, y, v);  // by all lanes: the exchange reads its partners' registers
      if (i >= a.I || left <= 0) continue;
      if (a.splits > 1) {
        const int64_t plane = PAIRED && AMAJ ? (int64_t)split * 2 + second : (int64_t)split;
        float* p = a.part + (plane * a.I + i) * a.Jp + j;  // Jp: J rounded up to 8
        *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += b[k];
        finish<BF, EPI>(a, out, i, j, left, v, res[x]);
      }
    }
  }
}

// Adds the partial products of a split in their order and finishes 8 outputs a lane, in `groups` workgroups.
// The workgroups after those add up db's partial sums, 16 columns each, 16 rows at a time: one launch where
// two would follow each other.
template <bool BF, int EPI>
__global__ void __launch_bounds__(256) linear_join_kernel(LinearArgs a, int groups) {
  if ((int)blockIdx.x >= groups) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int64_t i = (int64_t)((int)blockIdx.x - groups) * 16 + c;
    float s = 0.0f;
    if (i < a.I) {
#pragma unroll 4
      for (int p = r; p < a.db_parts; p += 16) s += a.db_part[p * a.I + i];
    }
    sums[r][c] = s;
    __syncthreads();
    if (r == 0 && i < a.I) {
      s = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) s += sums[k][c];
      static_cast<uint16_t*>(a.db)[i] = (uint16_t)pack2(s, 0.0f, BF);
    }
    return;
  }
  const int64_t per = a.Jp / 8, rows = a.y2 ? 2 * a.I : a.I, n = rows * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)groups * 256) {
    const int64_t i = t / per, j = (t - i * per) * 8;
    const float* p = a.part + i * a.Jp + j;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);
    if (EPI != kNoEpilogue && a.bias) load16(v, a.bias, j, left, BF);
    f32x4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      s0 += *reinterpret_cast<const f32x4_t*>(p + s * rows * a.Jp);
      s1 += *reinterpret_cast<const f32x4_t*>(p + s * rows * a.Jp + 4);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] += s0[k];
      v[4 + k] += s1[k];
    }
    const u32x4_t res = EPI != kNoEpilogue && a.res ? load_raw(a.res, i * a.sres + j, left) : u32x4_t{0u, 0u, 0u, 0u};
    finish<BF, EPI>(a, i < a.I ? a.y : a.y2, i < a.I ? i : i - a.I, j, left, v, res);
  }
}

// Forward of few rows (up to 16 MF): a workgroup computes 16 outputs of all rows, its eight waves take every
// eighth k-step of 32 each, straight from memory to registers: W is read once, by N / 16 workgroups,
// with all loads of a wave in flight, where a tile would wait for its stages one by one. The waves' sums meet in
// LDS in the waves' order.
template <bool BF, int MF>
__global__ void __launch_bounds__(512) linear_few_kernel(LinearArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[8][MF][256];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t j0 = (int64_t)blockIdx.x * 16;
  // rows past the end read the last one again; what comes of them is not stored
  const int last = (int)(a.J - 1 - j0), jr = c < last ? c : last;
  const rsrc_t rw = make_rsrc(static_cast<const uint16_t*>(a.B) + j0 * a.sb, 0x7fffffffu);
  const rsrc_t rx = make_rsrc(a.A, 0x7fffffffu);
  const uint32_t ow = (uint32_t)(jr * a.sb * 2);
  uint32_t ox[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) ox[f] = (uint32_t)((f * 16 + c < a.I ? f * 16 + c : a.I - 1) * a.sa * 2);
  f32x4_t acc[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // k-steps in flight
  const int K = (int)a.K;
  for (int k0 = wave * 32; k0 < K; k0 += U * 256) {
    u32x4_t vw[U], vx[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 256 + g * 8;  // chunks past K read as zeros
      vw[u] = ld16(rw, k < K ? ow + 2 * k : kOOB);
#pragma unroll
      for (int f = 0; f < MF; ++f) vx[u][f] = ld16(rx, k < K ? ox[f] + 2 * k : kOOB);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) acc[f] = mfma16x16x32<BF>(vw[u], vx[u][f], acc[f]);
  }
  // lane (c, g) holds outputs j0 + 4 g .. + 3 of row c
#pragma unroll
  for (int f = 0; f < MF; ++f) *reinterpret_cast<f32x4_t*>(&sums[wave][f][c * 16 + 4 * g]) = acc[f];
  __syncthreads();
  if (threadIdx.x < MF * 32) {
    const int f = threadIdx.x >> 5, at = (threadIdx.x & 31) * 8;  // 8 outputs of a row
    const int64_t i = f * 16 + at / 16, j = j0 + at % 16;
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);
    if (i < a.I && left > 0) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
      if (a.bias) load16(v, a.bias, j, left, BF);
      const u32x4_t res = a.res ? load_raw(a.res, i * a.sres + j, left) : u32x4_t{0u, 0u, 0u, 0u};
      f32x4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        s0 += *reinterpret_cast<const f32x4_t*>(&sums[u][f][at]);
        s1 += *reinterpret_cast<const f32x4_t*>(&sums[u][f][at + 4]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] += s0[k];
        v[4 + k] += s1[k];
      }
      finish<BF, kAnyAct>(a, a.y, i, j, left, v, res);
    }
  }
}

// dz = dy act'(z) in 16 bits (rows padded with zeros to Np), from the forward's slopes, and the column sums of the
// unrounded dz over each workgroup's rows. A lane holds 8 columns; a row takes as few lanes as hold it (up to
// 64), so a workgroup takes 256 / lanes rows at a time.
// WHOLE: N is a multiple of 8, no lane's columns end early (the code for those in the loop costs all rows 15 %).
template <bool BF, bool WHOLE>
__global__ void __launch_bounds__(256) linear_dz_kernel(DzArgs a) {
  __shared__ float sums[256 * 9];
  const int lanes = a.lanes, rows = 256 / lanes, lane = threadIdx.x & (lanes - 1), row = threadIdx.x / lanes;
  const int64_t j0 = (int64_t)blockIdx.x * lanes * 8, j = j0 + lane * 8;
  const int left = WHOLE ? 8 : (int)(a.N - j < 0 ? 0 : a.N - j < 8 ? a.N - j : 8);
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.0f;
  if (j < a.Np) {
    for (int64_t i = (int64_t)blockIdx.y * rows + row; i < a.M; i += (int64_t)gridDim.y * rows) {
      float v[8];
      load16(v, a.dy, i * a.sdy + j, left, BF);
      if (a.slope) {
        const u32x4_t w = load_raw(a.slope, i * a.N + j, left);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t x = w[k / 2];
          v[k] *= slope_of<BF>((k & 1) ? x >> 16 : x & 0xffffu);
        }
      }
      if (a.dz) store16(a.dz, i * a.Np + j, 8, v, BF);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += v[k];
    }
  }
  if (!a.part) return;
  // column k of a lane at a pitch of 9: the lanes' writes fall in different banks
#pragma unroll
  for (int k = 0; k < 8; ++k) sums[threadIdx.x * 9 + k] = s[k];
  __syncthreads();
  for (int c = threadIdx.x; c < lanes * 8; c += 256) {
    float t = 0.0f;
    for (int r = 0; r < rows; ++r) t += sums[(r * lanes + c / 8) * 9 + c % 8];
    if (j0 + c < a.N) a.part[(int64_t)blockIdx.y * a.N + j0 + c] = t;
  }
}

// Gradients of no rows: n zeros of 16 bits, 8 a lane at a time.
__global__ void __launch_bounds__(256) linear_zero_kernel(void* out, int64_t n) {
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; at < n; at += (int64_t)gridDim.x * 256 * 8)
    store_raw(out, at, (int)(n - at < 8 ? n - at : 8), u32x4_t{0u, 0u, 0u, 0u});
}

template <bool BF, bool AMAJ, bool BMAJ, int WI, int WJ, int FI, int FJ, int NS, int EPI, bool PAIRED>
void run(const LinearArgs& a, int64_t grid, hipStream_t s) {
  linear_kernel<BF, AMAJ, BMAJ, WI, WJ, FI, FJ, NS, EPI, PAIRED><<<(unsigned)grid, WI * WJ * 64, 0, s>>>(a);
}

template <bool BF>
hipError_t launch_few(const LinearArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((a.J + 15) / 16);
  switch ((a.I + 15) / 16) {
    case 1: linear_few_kernel<BF, 1><<<grid, 512, 0, s>>>(a); break;
    case 2: linear_few_kernel<BF, 2><<<grid, 512, 0, s>>>(a); break;
    case 3: linear_few_kernel<BF, 3><<<grid, 512, 0, s>>>(a); break;
    default: linear_few_kernel<BF, 4><<<grid, 512, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <bool BF, bool AMAJ, bool BMAJ, int EPI, bool PAIRED = false>
void run_tile(const LinearArgs& a, int tile, int64_t grid, hipStream_t s) {
  switch (tile) {
    case kTile256: return run<BF, AMAJ, BMAJ, 2, 4, 8, 4, 2, EPI, PAIRED>(a, grid, s);
    case kTile128: return run<BF, AMAJ, BMAJ, 2, 2, 4, 4, 2, EPI, PAIRED>(a, grid, s);
    case kTile128Deep: return run<BF, AMAJ, BMAJ, 2, 2, 4, 4, 4, EPI, PAIRED>(a, grid, s);
    default: return run<BF, AMAJ, BMAJ, 2, 2, 2, 2, 4, EPI, PAIRED>(a, grid, s);
  }
}

template <bool BF, bool AMAJ, bool BMAJ, bool FORWARD>
hipError_t launch(const LinearArgs& a, int tile, hipStream_t s) {
  const int64_t grid = a.ti * a.tj * a.splits;
  constexpr int kJoin = FORWARD ? kAnyAct : kNoEpilogue;
  if constexpr (!FORWARD) {
    bool done = false;
    if constexpr (BMAJ) {
      if (a.B2 || a.y2) {
        run_tile<BF, AMAJ, BMAJ, kNoEpilogue, true>(a, tile, grid, s);
        done = true;
      }
    }
    if (!done) run_tile<BF, AMAJ, BMAJ, kNoEpilogue>(a, tile, grid, s);
  } else {
    switch (a.splits == 1 ? a.act : FMX_ACT_NONE) {  // parts of k: the second kernel has the epilogue
      case FMX_ACT_RELU: run_tile<BF, AMAJ, BMAJ, FMX_ACT_RELU>(a, tile, grid, s); break;
      case FMX_ACT_GELU: run_tile<BF, AMAJ, BMAJ, FMX_ACT_GELU>(a, tile, grid, s); break;
      case FMX_ACT_GELU_TANH: run_tile<BF, AMAJ, BMAJ, FMX_ACT_GELU_TANH>(a, tile, grid, s); break;
      case FMX_ACT_SILU: run_tile<BF, AMAJ, BMAJ, FMX_ACT_SILU>(a, tile, grid, s); break;
      default: run_tile<BF, AMAJ, BMAJ, FMX_ACT_NONE>(a, tile, grid, s); break;
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t need = ((a.y2 ? 2 * a.I : a.I) * (a.Jp / 8) + 255) / 256;
  const int groups = (int)(need < 4096 ? need : 4096);
  linear_join_kernel<BF, kJoin><<<groups + (a.db ? (int)((a.I + 15) / 16) : 0), 256, 0, s>>>(a, groups);
  return hipGetLastError();
}

}  // namespace

// Time of a product by tile and split, in us, from times measured on one MI355X: a stage of 64 k with a compute unit's
// workgroups alone and all there, and what a tile costs besides (first loads, epilogue). Sizes that take it
// the other way, measured / by this rule (bf16):
//   16384 x 4096, k 1024: 256 tiles 132 / 127, 128 tiles 158 / 158      8192 x 1024, k 4096: 128 tiles 62 / 69, 256 99 / 101
//   24576 x 128, k 2048: 128 deep 34 / 23 (bound by HBM), 64 45 / 30    2048 x 1024, k 1024: 64 tiles 10 / 10, 128 16 / 16
//   128 x 2048, k 24576: 128 deep in 16 parts 33 / 25, 128 in 32 36 / 27
//   1024 x 4096, k 7777: 256 in 4 parts 69 / 73, 128 deep 84 / 75, 128 in 2 85 / 76
struct TileCost {
  int tile, size, per_cu;
  double alone, full, rest;
};
constexpr TileCost kCosts[] = {{kTile256, 256, 1, 1.45, 1.45, 8.5},
                               {kTile128, 128, 2, 0.75, 1.02, 3.4},
                               {kTile128Deep, 128, 1, 0.58, 0.58, 4.0},
                               {kTile64, 64, 2, 0.33, 0.43, 3.0}};

LinearPlan linear_plan(LinearForm form, int64_t I, int64_t J, int64_t K, bool pair) {
  const int64_t cus = layer_cus();
  static constexpr int kParts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  static constexpr int kPairParts[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 24};
  LinearPlan best = {};
  // Few rows straight from memory: every workgroup reads all of x, which costs more than the tiles' waits once
  // x is large (us, few / tiles; 32 x 768 -> 128 4.4 / 7.0, 64 x 1024 -> 4096 7.4 / 9.6, 16 x 4096 -> 1024 9.6 / 9.1,
  // 32 x 2048 -> 128 7.6 / 7.5, 64 x 4096 -> 1024 20 / 11).
  if (form == kLinearForward && I <= 64 && (I + 15) / 16 * K <= 4096) {
    best.tile = kFewRows;
    best.splits = 1;
    return best;
  }
  double least = 0;
  for (const TileCost& c : kCosts) {
    // The rows of a K-major tile are reached by 32-bit offsets below 2^31 from its first one. x and W have strides
    // below 2^22, which all tiles hold; dz has N's, below 2^24: tiles of 256 rows to N = 4.2 million, of 128 to 8.4.
    if (form != kLinearWeight && (c.size - 1) * K * 2 + BK * 2 > 0x7fffffff) continue;
    const int64_t ti = (I + c.size - 1) / c.size * (pair ? 2 : 1), tj = (J + c.size - 1) / c.size, slots = cus * c.per_cu;
    for (int want : pair ? kPairParts : kParts) {
      int64_t per = ((K + want - 1) / want + BK - 1) / BK * BK;
      if (want > 1 && per < 4 * BK) break;  // a part shorter than its loads' latency
      const int64_t splits = (K + per - 1) / per, n = ti * tj * splits, whole = n / slots, left = n % slots;
      const double stages = (double)((per + BK - 1) / BK);
      double us = whole * (stages * c.full + c.rest);
      if (left) us += stages * (left > cus ? c.full : c.alone) + c.rest;
      // partial products written and read, mostly in the caches, and the second kernel
      if (splits > 1) us += 2.5 + (double)splits * (double)I * (double)J * (pair ? 16.0 : 8.0) / 8e6;
      if (best.splits == 0 || us < least) {
        least = us;
        best.tile = c.tile;
        best.size = c.size;
        best.splits = (int)splits;
        best.ti = ti;
        best.tj = tj;
        best.split_k = per;
      }
    }
  }
  // Tile rows walked together: 1024 rows of the output, over as many columns as are on the GPU at once (us, 4 / 8
  // tile rows; 128 tiles 7777 x 1024 from k 4096 77.5 / 71.8, 256 tiles 16384 x 4096 with z 198 / 210).
  best.band = 1024 / best.size;
  return best;
}

size_t linear_part_bytes(const LinearPlan& p, int64_t I, int64_t J, bool pair) {
  return p.splits > 1 ? (pair ? 2 : 1) * (size_t)p.splits * (size_t)I * (size_t)((J + 7) / 8 * 8) * sizeof(float) : 0;
}

hipError_t launch_linear(bool bf16, LinearForm form, LinearArgs a, const LinearPlan& p, hipStream_t s) {
  // a launch has fewer than 2^32 threads: more rows than this go in several (their tiles fill the GPU, so k is whole)
  constexpr int64_t kRows = (int64_t)1 << 24;
  if (form != kLinearWeight && a.I > kRows && p.splits == 1) {
    for (int64_t at = 0; at < a.I; at += kRows) {
      LinearArgs b = a;
      b.I = a.I - at < kRows ? a.I - at : kRows;
      b.A = static_cast<const uint16_t*>(a.A) + at * a.sa;
      b.y = static_cast<uint16_t*>(a.y) + at * a.J;
      if (a.slope) b.slope = static_cast<int16_t*>(a.slope) + at * a.J;
      if (a.res) b.res = static_cast<const uint16_t*>(a.res) + at * a.sres;
      LinearPlan q = p;
      q.ti = (b.I + p.size - 1) / p.size;
      const hipError_t e = launch_linear(bf16, form, b, q, s);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  a.ti = p.ti;
  a.tj = p.tj;
  a.splits = p.splits;
  a.split_k = p.split_k;
  a.band = p.band;
  a.Jp = (a.J + 7) / 8 * 8;
  a.Jr = form == kLinearForward ? a.J : a.Jp;  // row-major B: whole chunks of 8 columns
  if (a.y2) a.half = (int)(p.ti / 2);
  if (p.tile == kFewRows) return bf16 ? launch_few<true>(a, s) : launch_few<false>(a, s);
  switch (form) {
    case kLinearForward:
      return bf16 ? launch<true, false, false, true>(a, p.tile, s) : launch<false, false, false, true>(a, p.tile, s);
    case kLinearInput:
      return bf16 ? launch<true, false, true, false>(a, p.tile, s) : launch<false, false, true, false>(a, p.tile, s);
    default:
      return bf16 ? launch<true, true, true, false>(a, p.tile, s) : launch<false, true, true, false>(a, p.tile, s);
  }
}

namespace {
int dz_lanes(int64_t N) {
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < N) lanes *= 2;
  return lanes;
}
}  // namespace

int linear_dz_parts(int64_t M, int64_t N) {
  const int64_t lanes = dz_lanes(N), rows = 256 / lanes, cols = (N + lanes * 8 - 1) / (lanes * 8);
  int64_t parts = (int64_t)layer_cus() * 8 / cols;      // about eight workgroups a CU
  if (parts > 256) parts = 256;                         // rows that the second kernel adds
  const int64_t most = (M + rows * 2 - 1) / (rows * 2);  // two rows a thread at least
  if (parts > most) parts = most;
  return (int)(parts < 1 ? 1 : parts);
}

hipError_t launch_linear_dz(bool bf16, DzArgs a, int parts, hipStream_t s) {
  a.lanes = dz_lanes(a.N);
  // without the sums to hold them together, the rows go to as many workgroups as they fill
  const int64_t rows = 4 * 256 / a.lanes, most = (a.M + rows - 1) / rows;
  const int64_t y = a.part ? parts : most < 65535 ? most : 65535;
  const dim3 grid((unsigned)((a.Np + a.lanes * 8 - 1) / (a.lanes * 8)), (unsigned)y);
  if (a.N % 8 == 0) {
    if (bf16)
      linear_dz_kernel<true, true><<<grid, 256, 0, s>>>(a);
    else
      linear_dz_kernel<false, true><<<grid, 256, 0, s>>>(a);
  } else if (bf16) {
    linear_dz_kernel<true, false><<<grid, 256, 0, s>>>(a);
  } else {
    linear_dz_kernel<false, false><<<grid, 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_linear_zero(void* out, int64_t n, hipStream_t s) {
  const int64_t need = (n + 2047) / 2048, most = (int64_t)layer_cus() * 8;
  linear_zero_kernel<<<(unsigned)(need < most ? need : most), 256, 0, s>>>(out, n);
  return hipGetLastError();
}

}  // namespace fmx
