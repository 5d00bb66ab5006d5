// Gated linear layer on MFMA: y = act(x Wg^T + bg) * (x Wu^T + bu), and the first pass of its backward.
//
// One tile of x meets the rows of both weights that make the same outputs: a workgroup holds TI x TJ sums of
// either product, a lane both values of each of its outputs, so the activation and the product need no pass of
// their own and neither product reaches memory. Stages and fragments are those of the linear layer (a tile of
// 256 rows x 128 outputs moves and multiplies what its 256 x 256 tile does).
//
// The backward is, with g and u the two products,
//   dg = dy u act'(g),  du = dy act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// The forward keeps the factors u act'(g) and act(g) (see FactorCode), so that the backward needs no
// exponentials and no products again; its first pass writes dg and du beside each other, [M, 2 Np], and
// dx is one product over both, the weights taking turns.
//
// Bound by MFMA and power where rows are many: 8192 x 1024 -> 4096 with SiLU, bf16, 110-124 us by clock (1.2 PFLOP/s; the library's
// plain products of those sizes 1.25). A training step of 16384 x 1024 -> 2816 655-680: forward 214-254 (276 MB of y and
// factors), dz 80 (450 MB, 5.6 TB/s), dx 171-193, dw 198-235 and its join 21. Bound by the launch where they are few: 32 x 768 -> 1152
// 5.9 a call.
#include "fmx_device.h"
#include "fmx_layers.h"
#include "fmx_product.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

// ---- the factors between the passes ----

// A factor kept in the operands' type would be rounded twice before it is multiplied (with dg itself): gradients 1.73
// times as far from 64 bits as ones rounded once, where dg's and the result's roundings alone make 1.41. So it is kept
// with more bits than they have:
//   bf16  16 bits: sign, and a measure of |v|'s logarithm (its float32 bits) in steps of 2^-9 of a power of two from 2^-16
//         to 2^16, of 2^-7 from there down to 2^-80 and up to 2^79.9: off by 2^-10 (2^-8) of the factor at most, 1.44
//         times. 0 is exact, what is smaller than 2^-80 becomes 0, what is larger than 2^79.9 and NaN: NaN.
//   fp16  24 bits: float32 without its last 8, off by 2^-16: 1.41 times. The low bytes of both factors make a plane
//         of their own.
template <bool BF>
struct FactorCode {
  // The three lines meet where the steps change: a code's value is the middle one of them, and so is a value's code.
  static constexpr int kLow = (127 - 16) << 23, kHigh = (127 + 16) << 23;
  static constexpr int kFine = (kLow >> 14) - 8192, kBelow = (kLow >> 16) - 8192, kAbove = (kHigh >> 16) - 24576;
  static __device__ __forceinline__ int middle(int below, int fine, int above) {
    const int v = fine < above ? fine : above;
    return v > below ? v : below;  // below < above
  }
  static __device__ __forceinline__ uint32_t encode(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    if constexpr (!BF) return b + 0x80u;  // its upper 24 bits
    const uint32_t m = b & 0x7fffffffu;
    const int coarse = (int)((m + 0x8000u) >> 16);
    int c = middle(coarse - kBelow, (int)((m + 0x2000u) >> 14) - kFine, coarse - kAbove);
    c = c > 0 ? c : 0;
    c = c < 32767 ? c : 32767;
    return (uint32_t)c | ((b >> 16) & 0x8000u);
  }
  static __device__ __forceinline__ float decode(uint32_t hi, uint32_t lo) {
    if constexpr (!BF) return __builtin_bit_cast(float, (hi << 16) | (lo << 8));
    const int c = (int)(hi & 0x7fffu);
    // The lines the other way round: the coarse ones are the steeper. The one of small values passes 2^31 and is negative
    // from code 26752 on; the middle one is that of large values there all the same.
    uint32_t m = (uint32_t)middle((c + kAbove) * 65536, (c + kFine) * 16384, (int)((uint32_t)(c + kBelow) << 16));
    m = c == 0 ? 0u : c == 32767 ? 0x7fc00000u : m;
    return __builtin_bit_cast(float, m | ((hi & 0x8000u) << 16));
  }
};

// The codes of 8 neighbouring pairs of factors, as 16-byte pieces of the planes.
template <bool BF>
struct Factors8 {
  u32x4_t g, u, lo;
  __device__ __forceinline__ Factors8(const float (&fg)[8], const float (&fu)[8]) {
    lo = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = FactorCode<BF>::encode(fg[2 * k]), b = FactorCode<BF>::encode(fg[2 * k + 1]);
      const uint32_t c = FactorCode<BF>::encode(fu[2 * k]), d = FactorCode<BF>::encode(fu[2 * k + 1]);
      if constexpr (BF) {
        g[k] = a | (b << 16);
        u[k] = c | (d << 16);
      } else {
        g[k] = (a >> 16) | (b & 0xffff0000u);
        u[k] = (c >> 16) | (d & 0xffff0000u);
        lo[k] = ((a >> 8) & 0xffu) | (c & 0xff00u) | ((b & 0xff00u) << 8) | ((d & 0xff00u) << 16);
      }
    }
  }
};

// act(g) of 8 outputs (biases added), and with KEEP dg's factor in g's place. (The product with u is left to the
// caller, in one form: it may be rounded to 16 bits together with its own rounding, and y has the same bits with and
// without KEEP.)
template <int ACT, bool KEEP>
__device__ __forceinline__ void gate8(float (&g)[8], const float (&u)[8], float (&y)[8], int act) {
  if constexpr (ACT >= 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float slope;
      y[k] = act_value<KEEP>(g[k], ACT, slope);
      if constexpr (KEEP) g[k] = u[k] * slope;
    }
  } else {
    switch (act) {  // uniform: one test for the eight
      case FMX_ACT_RELU: gate8<FMX_ACT_RELU, KEEP>(g, u, y, act); break;
      case FMX_ACT_GELU: gate8<FMX_ACT_GELU, KEEP>(g, u, y, act); break;
      case FMX_ACT_GELU_TANH: gate8<FMX_ACT_GELU_TANH, KEEP>(g, u, y, act); break;
      case FMX_ACT_SILU: gate8<FMX_ACT_SILU, KEEP>(g, u, y, act); break;
      default: gate8<FMX_ACT_NONE, KEEP>(g, u, y, act); break;
    }
  }
}
__device__ __forceinline__ u32x4_t product8(const float (&a)[8], const float (&u)[8], bool bf) {
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = a[k] * u[k];
  return pack8(y, bf);
}

__device__ __forceinline__ void add_bias(float (&v)[8], const void* bias, int64_t j, int left, bool bf) {
  if (!bias) return;
  float b[8];
  load16(b, bias, j, left, bf);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += b[k];
}

// 8 outputs j .. j + 7 of row i, of which `left` exist: from the two products to memory.
template <bool BF, int ACT>
__device__ __forceinline__ void finish(const GatedArgs& a, int64_t i, int64_t j, int left, float (&g)[8], float (&u)[8]) {
  const int64_t at = i * a.J + j;
  float y[8];
  if (a.keep) {
    gate8<ACT, true>(g, u, y, a.act);
    const Factors8<BF> f(g, y);
    const int64_t plane = a.I0 * a.J;
    store_raw(a.keep, at, left, f.g);
    store_raw(a.keep, plane + at, left, f.u);
    if constexpr (!BF) store_raw(a.keep, 2 * plane + at, left, f.lo);
  } else {
    gate8<ACT, false>(g, u, y, a.act);
  }
  store_raw(a.y, at, left, product8(y, u, BF));
}

// ---- tiles ----

template <bool BF, int WI, int WJ, int FI, int FJ, int NS, int ACT>
__global__ void __launch_bounds__(WI* WJ * 64) gated_kernel(GatedArgs a) {
  constexpr int TI = WI * FI * 16, TJ = WJ * FJ * 16, NT = WI * WJ * 64;
  constexpr int AT_G = TI * BK * 2, AT_U = AT_G + TJ * BK * 2, BYTES = AT_U + TJ * BK * 2;
  using SideA = Side<false, false, TI, NT>;
  using SideB = Side<false, true, TJ, NT>;
  constexpr int LOADS = SideA::kLoads + 2 * SideB::kLoads;
  __shared__ __attribute__((aligned(1024))) unsigned char lds0[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds1[BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char lds2[NS > 2 ? BYTES : 16];
  __shared__ __attribute__((aligned(1024))) unsigned char lds3[NS > 2 ? BYTES : 16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave % WI, wj = wave / WI;
  const Place at(blockIdx.x, (uint32_t)a.ti, (uint32_t)a.tj, (uint32_t)a.splits, (uint32_t)a.band);
  const int64_t i0 = (int64_t)at.row * TI, j0 = (int64_t)at.col * TJ;
  const int64_t k0 = (int64_t)at.split * a.split_k;
  const int64_t kn = a.K - k0 < a.split_k ? a.K - k0 : a.split_k;
  const int nit = (int)((kn + BK - 1) / BK);

  const SideA sa(a.x, a.sx, i0, a.I, k0, tid);
  const SideB sg(a.wg, a.swg, j0, a.J, k0, tid), su(a.wu, a.swu, j0, a.J, k0, tid);
  const Frags<false, false, TI> fa(wi * FI * 16, lane);
  const Frags<false, true, TJ> fb(wj * FJ * 16, lane);

  f32x4_t ag[FI][FJ], au[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) ag[x][y] = au[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};

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
    sg.issue(lds + AT_G, it, left, wave);
    su.issue(lds + AT_U, it, left, wave);
  };
  u32x4_t va[2][FI], vg[2][FJ], vu[2][FJ];
  auto read = [&](auto set, const unsigned char* lds, int kk) __attribute__((always_inline)) {
    constexpr int Z = decltype(set)::value;
#pragma unroll
    for (int y = 0; y < FJ; ++y) vg[Z][y] = fb.read(lds + AT_G, y, kk);
#pragma unroll
    for (int y = 0; y < FJ; ++y) vu[Z][y] = fb.read(lds + AT_U, y, kk);
#pragma unroll
    for (int x = 0; x < FI; ++x) va[Z][x] = fa.read(lds, x, kk);
  };
  auto multiply = [&](auto set) __attribute__((always_inline)) {
    constexpr int Z = decltype(set)::value;
#pragma unroll
    for (int x = 0; x < FI; ++x) {
#pragma unroll
      for (int y = 0; y < FJ; ++y) ag[x][y] = mfma16x16x32<BF>(vg[Z][y], va[Z][x], ag[x][y]);
#pragma unroll
      for (int y = 0; y < FJ; ++y) au[x][y] = mfma16x16x32<BF>(vu[Z][y], va[Z][x], au[x][y]);
    }
  };
  run_stages<NS, LOADS, 2 * FJ + FI, 2 * FI * FJ>(nit, buffer, issue, read, multiply, [](auto) {});

  // A lane holds row c of each i fragment, and of a pair of j fragments 8 consecutive outputs of either product.
  const int c = lane & 15, g = lane >> 4;
  auto pair = [&](const f32x4_t (&acc)[FI][FJ], int x, int y, float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = acc[x][y][k];
      v[4 + k] = acc[x][y + 1][k];
    }
  };
  if (FJ == 4 && a.splits == 1 && i0 + TI <= a.I && j0 + TJ <= a.J) {
    // A whole tile: a wave turns its 16 x 64 blocks into rows of 128 bytes, whole lines of memory, in LDS
    // that nothing is read from or loaded into any more.
    stage_barrier();
    unsigned char* mine = (wave < WI * WJ / 2 ? lds0 : lds1) + (wave % (WI * WJ / 2)) * (BYTES / (WI * WJ / 2));
    static_assert(FJ != 4 || BYTES / (WI * WJ / 2) >= FI * 2048, "a wave's blocks");
    const int64_t jw = j0 + wj * FJ * 16;
    float bg[2][8], bu[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 8; ++k) bg[h][k] = bu[h][k] = 0.0f;
      add_bias(bg[h], a.bg, jw + 32 * h + 8 * g, 8, BF);
      add_bias(bu[h], a.bu, jw + 32 * h + 8 * g, 8, BF);
    }
    const int row = lane >> 3, ch = lane & 7;
    const int64_t plane = a.I0 * a.J;
    auto put = [&](int x, int h, const u32x4_t& w) __attribute__((always_inline)) {
      *reinterpret_cast<u32x4_t*>(mine + x * 2048 + c * 128 + (((4 * h + g) ^ (c & 7)) << 4)) = w;
    };
    auto flush = [&](int x, void* out, int64_t from) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(mine + x * 2048 + (row + 8 * h) * 128 + ((ch ^ row) << 4));
        const int64_t i = i0 + wi * FI * 16 + x * 16 + row + 8 * h;
        store_raw(out, from + i * a.J + jw + ch * 8, 8, w);
      }
    };
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      float vg8[2][8], vu8[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pair(ag, x, 2 * h, vg8[h]);
        pair(au, x, 2 * h, vu8[h]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          vg8[h][k] += bg[h][k];
          vu8[h][k] += bu[h][k];
        }
      }
      float y[2][8];
      if (a.keep) {
        u32x4_t fu[2], lo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          gate8<ACT, true>(vg8[h], vu8[h], y[h], a.act);
          const Factors8<BF> f(vg8[h], y[h]);
          put(x, h, f.g);
          fu[h] = f.u;
          lo[h] = f.lo;
        }
        flush(x, a.keep, 0);
        put(x, 0, fu[0]);
        put(x, 1, fu[1]);
        flush(x, a.keep, plane);
        if constexpr (!BF) {
          put(x, 0, lo[0]);
          put(x, 1, lo[1]);
          flush(x, a.keep, 2 * plane);
        }
      } else {
        gate8<ACT, false>(vg8[0], vu8[0], y[0], a.act);
        gate8<ACT, false>(vg8[1], vu8[1], y[1], a.act);
      }
      put(x, 0, product8(y[0], vu8[0], BF));
      put(x, 1, product8(y[1], vu8[1], BF));
      flush(x, a.y, 0);
    }
    return;
  }
#pragma unroll
  for (int y = 0; y < FJ; y += 2) {
    const int64_t j = j0 + wj * FJ * 16 + y * 16 + 8 * g;
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);  // columns inside; none: nothing is stored
    if (left <= 0) continue;
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      const int64_t i = i0 + wi * FI * 16 + x * 16 + c;
      if (i >= a.I) continue;
      float v[8], u[8];
      pair(ag, x, y, v);
      pair(au, x, y, u);
      if (a.splits > 1) {
        float* p = a.part + (((int64_t)at.split * 2) * a.I + i) * a.Jp + j;  // Jp: J rounded up to 8
        *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
        p += a.I * a.Jp;
        *reinterpret_cast<f32x4_t*>(p) = f32x4_t{u[0], u[1], u[2], u[3]};
        *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{u[4], u[5], u[6], u[7]};
      } else {
        add_bias(v, a.bg, j, left, BF);
        add_bias(u, a.bu, j, left, BF);
        finish<BF, ACT>(a, i, j, left, v, u);
      }
    }
  }
}

// Adds the partial products of a split in their order and finishes 8 outputs a lane.
template <bool BF>
__global__ void __launch_bounds__(256) gated_join_kernel(GatedArgs a) {
  const int64_t per = a.Jp / 8, n = a.I * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
    const int64_t i = t / per, j = (t - i * per) * 8, plane = a.I * a.Jp;
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);
    const float* p = a.part + i * a.Jp + j;
    f32x4_t s[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) s[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) s[q] += *reinterpret_cast<const f32x4_t*>(p + (2 * k + q / 2) * plane + 4 * (q & 1));
    float v[8], u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = s[k / 4][k % 4];
      u[k] = s[2 + k / 4][k % 4];
    }
    add_bias(v, a.bg, j, left, BF);
    add_bias(u, a.bu, j, left, BF);
    finish<BF, kAnyAct>(a, i, j, left, v, u);
  }
}

// Few rows (up to 16 MF): a workgroup computes 16 outputs of all rows, its eight waves take every eighth k-step of 32
// each, straight from memory to registers, with all loads of a wave in flight. The waves' sums meet in LDS in the
// waves' order.
template <bool BF, int MF>
__global__ void __launch_bounds__(512) gated_few_kernel(GatedArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[8][2][MF][256];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t j0 = (int64_t)blockIdx.x * 16;
  // rows past the end read the last one again; what comes of them is not stored
  const int last = (int)(a.J - 1 - j0 < 15 ? a.J - 1 - j0 : 15), jr = c < last ? c : last;
  const rsrc_t rg = make_rsrc(static_cast<const uint16_t*>(a.wg) + j0 * a.swg, 0x7fffffffu);
  const rsrc_t ru = make_rsrc(static_cast<const uint16_t*>(a.wu) + j0 * a.swu, 0x7fffffffu);
  const rsrc_t rx = make_rsrc(a.x, 0x7fffffffu);
  const uint32_t og = (uint32_t)(jr * a.swg * 2), ou = (uint32_t)(jr * a.swu * 2);
  uint32_t ox[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) ox[f] = (uint32_t)((f * 16 + c < a.I ? f * 16 + c : a.I - 1) * a.sx * 2);
  f32x4_t ag[MF], au[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) ag[f] = au[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // k-steps in flight
  const int K = (int)a.K;
  for (int k0 = wave * 32; k0 < K; k0 += U * 256) {
    u32x4_t vg[U], vu[U], vx[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 256 + g * 8;  // chunks past K read as zeros
      vg[u] = ld16(rg, k < K ? og + 2 * k : kOOB);
      vu[u] = ld16(ru, k < K ? ou + 2 * k : kOOB);
#pragma unroll
      for (int f = 0; f < MF; ++f) vx[u][f] = ld16(rx, k < K ? ox[f] + 2 * k : kOOB);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        ag[f] = mfma16x16x32<BF>(vg[u], vx[u][f], ag[f]);
        au[f] = mfma16x16x32<BF>(vu[u], vx[u][f], au[f]);
      }
  }
  // lane (c, g) holds outputs j0 + 4 g .. + 3 of row c
#pragma unroll
  for (int f = 0; f < MF; ++f) {
    *reinterpret_cast<f32x4_t*>(&sums[wave][0][f][c * 16 + 4 * g]) = ag[f];
    *reinterpret_cast<f32x4_t*>(&sums[wave][1][f][c * 16 + 4 * g]) = au[f];
  }
  __syncthreads();
  if (threadIdx.x < MF * 32) {
    const int f = threadIdx.x >> 5, at = (threadIdx.x & 31) * 8;  // 8 outputs of a row
    const int64_t i = f * 16 + at / 16, j = j0 + at % 16;
    const int left = (int)(a.J - j < 8 ? a.J - j : 8);
    if (i < a.I && left > 0) {
      f32x4_t s[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) s[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += *reinterpret_cast<const f32x4_t*>(&sums[w][q / 2][f][at + 4 * (q & 1)]);
      float v[8], u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = s[k / 4][k % 4];
        u[k] = s[2 + k / 4][k % 4];
      }
      add_bias(v, a.bg, j, left, BF);
      add_bias(u, a.bu, j, left, BF);
      finish<BF, kAnyAct>(a, i, j, left, v, u);
    }
  }
}

// dg and du in 16 bits, [M, 2 Np] with zeros from N to Np, from dy and the forward's factors, and the column sums of
// both before rounding over each workgroup's rows. A lane holds 8 columns; a row takes as few lanes as hold it (up to
// 64), so a workgroup takes 256 / lanes rows at a time.
// WHOLE: N is a multiple of 8, no lane's columns end early.
template <bool BF, bool WHOLE>
__global__ void __launch_bounds__(256) gated_dz_kernel(GatedDzArgs a) {
  __shared__ float sums[256 * 9];
  const int lanes = a.lanes, rows = 256 / lanes, lane = threadIdx.x & (lanes - 1), row = threadIdx.x / lanes;
  const int64_t j0 = (int64_t)blockIdx.x * lanes * 8, j = j0 + lane * 8;
  const int left = WHOLE ? (j < a.N ? 8 : 0) : (int)(a.N - j < 0 ? 0 : a.N - j < 8 ? a.N - j : 8);
  const int64_t plane = a.M * a.N;
  float sg[8], su[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sg[k] = su[k] = 0.0f;
  if (j < a.Np) {
    for (int64_t i = (int64_t)blockIdx.y * rows + row; i < a.M; i += (int64_t)gridDim.y * rows) {
      float vg[8], vu[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) vg[k] = vu[k] = 0.0f;
      if (left > 0) {
        float dy[8];
        const int64_t at = i * a.N + j;
        const int n = WHOLE ? 8 : left;
        const u32x4_t y = load_raw(a.dy, i * a.sdy + j, n), g = load_raw(a.keep, at, n), u = load_raw(a.keep, plane + at, n);
        u32x4_t lo = {0u, 0u, 0u, 0u};
        if constexpr (!BF) lo = load_raw(a.keep, 2 * plane + at, n);
        unpack8(dy, y, BF);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t xg = g[k / 2], xu = u[k / 2], xl = lo[k / 2], sh = 16 * (k & 1);
          const float fg = FactorCode<BF>::decode((xg >> sh) & 0xffffu, (xl >> sh) & 0xffu);
          const float fu = FactorCode<BF>::decode((xu >> sh) & 0xffffu, (xl >> (sh + 8)) & 0xffu);
          if (WHOLE || k < left) {
            vg[k] = dy[k] * fg;
            vu[k] = dy[k] * fu;
          }
        }
      }
      if (a.dz) {
        store16(a.dz, i * 2 * a.Np + j, 8, vg, BF);
        store16(a.dz, i * 2 * a.Np + a.Np + j, 8, vu, BF);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sg[k] += vg[k];
        su[k] += vu[k];
      }
    }
  }
  if (!a.part) return;
  // column k of a lane at a pitch of 9: the lanes' writes fall in different banks
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[threadIdx.x * 9 + k] = half ? su[k] : sg[k];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * 8; c += 256) {
      float t = 0.0f;
      for (int r = 0; r < rows; ++r) t += sums[(r * lanes + c / 8) * 9 + c % 8];
      if (j0 + c < a.N) a.part[((int64_t)blockIdx.y * 2 + half) * a.N + j0 + c] = t;
    }
  }
}

template <bool BF, int ACT>
void run_tile(const GatedArgs& a, int tile, hipStream_t s) {
  const unsigned grid = (unsigned)(a.ti * a.tj * a.splits);
  switch (tile) {
    case kTile256: gated_kernel<BF, 4, 2, 4, 4, 2, ACT><<<grid, 512, 0, s>>>(a); break;
    case kTile192: gated_kernel<BF, 4, 1, 3, 4, 2, ACT><<<grid, 256, 0, s>>>(a); break;
    case kTile128: gated_kernel<BF, 2, 2, 4, 2, 2, ACT><<<grid, 256, 0, s>>>(a); break;
    case kTile128Deep: gated_kernel<BF, 2, 2, 4, 2, 4, ACT><<<grid, 256, 0, s>>>(a); break;
    default: gated_kernel<BF, 2, 2, 2, 2, 4, ACT><<<grid, 256, 0, s>>>(a); break;
  }
}

template <bool BF>
hipError_t launch(const GatedArgs& a, int tile, hipStream_t s) {
  if (tile == kFewRows) {
    const unsigned grid = (unsigned)((a.J + 15) / 16);
    switch ((a.I + 15) / 16) {
      case 1: gated_few_kernel<BF, 1><<<grid, 512, 0, s>>>(a); break;
      case 2: gated_few_kernel<BF, 2><<<grid, 512, 0, s>>>(a); break;
      case 3: gated_few_kernel<BF, 3><<<grid, 512, 0, s>>>(a); break;
      default: gated_few_kernel<BF, 4><<<grid, 512, 0, s>>>(a); break;
    }
    return hipGetLastError();
  }
  switch (a.splits == 1 ? a.act : FMX_ACT_NONE) {  // parts of k: the second kernel has the epilogue
    case FMX_ACT_RELU: run_tile<BF, FMX_ACT_RELU>(a, tile, s); break;
    case FMX_ACT_GELU: run_tile<BF, FMX_ACT_GELU>(a, tile, s); break;
    case FMX_ACT_GELU_TANH: run_tile<BF, FMX_ACT_GELU_TANH>(a, tile, s); break;
    case FMX_ACT_SILU: run_tile<BF, FMX_ACT_SILU>(a, tile, s); break;
    default: run_tile<BF, FMX_ACT_NONE>(a, tile, s); break;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t need = (a.I * (a.Jp / 8) + 255) / 256;
  gated_join_kernel<BF><<<(unsigned)(need < 4096 ? need : 4096), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// Time of a product by tile and split, as linear_plan's: rows and outputs of a tile, its stage with a compute unit's
// workgroups alone and all there, and what a tile costs besides.
struct GatedCost {
  int tile, rows, cols, per_cu;
  double alone, full, rest;
};
constexpr GatedCost kGatedCosts[] = {{kTile256, 256, 128, 1, 1.45, 1.45, 8.5},
                                     {kTile128, 128, 64, 2, 0.75, 1.02, 3.4},
                                     {kTile128Deep, 128, 64, 1, 0.58, 0.58, 4.0},
                                     {kTile64, 64, 64, 1, 0.40, 0.40, 3.0}};

GatedPlan gated_plan(int64_t I, int64_t J, int64_t K, bool keep) {
  const int64_t cus = layer_cus();
  GatedPlan best = {};
  if (I <= 64 && (I + 15) / 16 * K <= 4096) {  // as for the linear layer
    best.tile = kFewRows;
    best.splits = 1;
    return best;
  }
  double least = 0;
  for (const GatedCost& c : kGatedCosts) {
    const int64_t ti = (I + c.rows - 1) / c.rows, tj = (J + c.cols - 1) / c.cols, slots = cus * c.per_cu;
    for (int want : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const int64_t per = ((K + want - 1) / want + BK - 1) / BK * BK;
      if (want > 1 && per < 4 * BK) break;  // a part shorter than its loads' latency
      const int64_t splits = (K + per - 1) / per, n = ti * tj * splits, whole = n / slots, left = n % slots;
      const double stages = (double)((per + BK - 1) / BK);
      double us = whole * (stages * c.full + c.rest);
      if (left) us += stages * (left > cus ? c.full : c.alone) + c.rest;
      if (splits > 1) us += 2.5 + (double)splits * (double)I * (double)J * 16.0 / 8e6;
      if (best.splits == 0 || us < least) {
        least = us;
        best.tile = c.tile;
        best.splits = (int)splits;
        best.ti = ti;
        best.tj = tj;
        best.split_k = per;
        best.rows = c.rows;
        best.band = 1024 / c.rows;
      }
    }
  }
  // Where the factors are kept as well, three times the output, two workgroups a unit that cover each other's stores are
  // the better large tile (us, 256 x 128 / 192 x 64: training step 16384 x 1024 -> 2816 682 / 666, its forward alone
  // 208 / 209: the power saved goes to the products after it; 8192 x 1024 -> 4096 without factors 124 / 130; other training
  // steps 8192 x 1024 -> 4096 492 / 476, 32768 x 768 -> 2304 915 / 891, 32768 x 768 -> 1152 483 / 464, 4096 x 2048 -> 5632
  // 573 / 559, 65536 x 384 -> 1536 fp16 871 / 865, 8192 x 4096 -> 4096 1339 / 1358). The
  // tile alone changes, not the parts of k: y has the same bits with and without the factors.
  if (keep && best.tile == kTile256 && best.splits == 1) {
    best.tile = kTile192;
    best.rows = 192;
    best.ti = (I + 191) / 192;
    best.tj = (J + 63) / 64;
    best.band = 5;
  }
  return best;
}

size_t gated_part_bytes(const GatedPlan& p, int64_t I, int64_t J) {
  return p.splits > 1 ? (size_t)p.splits * 2 * (size_t)I * (size_t)((J + 7) / 8 * 8) * sizeof(float) : 0;
}

hipError_t launch_gated(bool bf16, GatedArgs a, const GatedPlan& p, hipStream_t s) {
  a.I0 = a.I;
  a.ti = p.ti;
  a.tj = p.tj;
  a.splits = p.splits;
  a.split_k = p.split_k;
  a.band = p.band;
  a.Jp = (a.J + 7) / 8 * 8;
  // a launch has fewer than 2^32 threads: more tiles than this go in several (they fill the GPU, so k is whole)
  constexpr int64_t kTiles = (int64_t)1 << 22;
  if (p.tile == kFewRows || p.splits > 1 || p.ti * p.tj <= kTiles)
    return bf16 ? launch<true>(a, p.tile, s) : launch<false>(a, p.tile, s);
  const int64_t rows = kTiles / p.tj * p.rows;
  for (int64_t at = 0; at < a.I0; at += rows) {
    GatedArgs b = a;
    b.I = a.I0 - at < rows ? a.I0 - at : rows;
    b.ti = (b.I + p.rows - 1) / p.rows;
    b.x = static_cast<const uint16_t*>(a.x) + at * a.sx;
    b.y = static_cast<uint16_t*>(a.y) + at * a.J;
    if (a.keep) b.keep = static_cast<uint16_t*>(a.keep) + at * a.J;  // the planes are I0 rows apart
    const hipError_t e = bf16 ? launch<true>(b, p.tile, s) : launch<false>(b, p.tile, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

namespace {
int dz_lanes(int64_t N) {
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < N) lanes *= 2;
  return lanes;
}
}  // namespace

int gated_dz_parts(int64_t M, int64_t N) { return linear_dz_parts(M, N); }

hipError_t launch_gated_dz(bool bf16, GatedDzArgs a, int parts, hipStream_t s) {
  a.lanes = dz_lanes(a.Np);
  // without the sums to hold them together, the rows go to as many workgroups as they fill
  const int64_t rows = 4 * 256 / a.lanes, most = (a.M + rows - 1) / rows;
  const int64_t y = a.part ? parts : most < 65535 ? most : 65535;
  const dim3 grid((unsigned)((a.Np + a.lanes * 8 - 1) / (a.lanes * 8)), (unsigned)y);
  if (a.N % 8 == 0) {
    if (bf16)
      gated_dz_kernel<true, true><<<grid, 256, 0, s>>>(a);
    else
      gated_dz_kernel<false, true><<<grid, 256, 0, s>>>(a);
  } else if (bf16) {
    gated_dz_kernel<true, false><<<grid, 256, 0, s>>>(a);
  } else {
    gated_dz_kernel<false, false><<<grid, 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace fmx
