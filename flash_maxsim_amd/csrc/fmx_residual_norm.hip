// The step from one block of an encoder to the next over rows of d elements: the block's output, normalised, gated and
// scaled, is added to the hidden states, and their norm is what the next block reads. Forward and backward.
//
//   norm(v) = (v - mu) s,  s = 1 / sqrt(mean (v - mu)^2 + eps),  mu = mean v (layer) or 0 (rms)
//   t = norm(x) pw + pb   (or x),   h = alpha r + scale gate t,   y = norm(h) w + b
// and with g = dh + s2 (wdy - mean(wdy) - hh mean(wdy hh)), wdy = w dy, hh = norm(h) (rms: without the first mean):
//   dr = alpha g,  dgate = g scale t,  q = g scale gate,  dx = s1 (q pw - mean(q pw) - xh mean(q pw xh)) (or q)
//   dw = sum dy hh,  db = sum dy,  dscale = sum g gate t,  dpw = sum q xh,  dpb = sum q   over the rows
//
// Bound by HBM: the forward reads x, r (and the gate) and writes h and y, once each; the backward reads x, r, the gate,
// dh and dy and writes dx, dr and dgate. y is the norm of h before its rounding, and the backward makes h anew from x
// and r rather than read the rounded one: the same bytes, and no gradient sees that rounding. Both norms' mu and s are
// kept, 16 bytes a row.
//
// A row lives in the registers of one to eight waves between its sums and its outputs, 8 elements a lane in the backward
// (its five column sums, four vectors of weights and two rows of five arrays spill at 16, which only rows of more than
// 4096 elements take) and up to 16 in the forward; a workgroup's eight waves walk the rows in strides of the launch, the
// next row (in the backward: the next two) loaded while this one is summed. Variances are those of centred values, from
// registers. Rows may begin at any element: accesses of 16 bytes need no more than an element's alignment here.
//
// 65536 x 1024 bf16 with both norms, gate and scale: forward 124 us (5.3 TB/s), backward 205 (5.2 TB/s; loads one row ahead
// 243, workgroups of four waves then 278), the join of its sums 5. 32 x 768: 3.9, a launch's own time. 65536 x 768 without a
// gate: fp16 82 and 147 us (4.9 and 4.1 TB/s: the backward's rows of 513 to 1023 columns have two waves with room for 1024), float32
// 154 and 224 (5.2 and 5.4 TB/s).
//
// Weight gradients: a workgroup adds its waves' sums in LDS in the waves' order and writes one row of partial sums; a
// second kernel adds those rows in a fixed order. No atomics. (The waves one after the other, in the columns' order with its
// bank conflicts, took 11 of 24 us of 1537 x 771 fp16; now 16.6.)
#include "fmx_device.h"
#include "fmx_layers.h"
#include "fmx_rows.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

constexpr int kWaves = 8;  // of a workgroup
constexpr int kThreads = kWaves * 64;

// Sums of a and of b over the NW waves that share a row, in every lane.
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

// Where a lane's elements lie: piece j of V elements at column ((j * NW + sub) * 64 + lane) * V, sub the wave's place
// among the NW of its row. WHOLE: d is a multiple of V, no piece ends early. Else the last piece begins at d - V and has some
// of the columns of the one before it: both lanes compute the same there and store the same, and `own` leaves them out of
// sums by a mask of a value's bits: a factor of zero would make NaN of an infinity. (Pieces that ended early, element by
// element: 65536 x 771 fp16, layer norms, forward 182 us, backward 355; with a factor 104 and 196, with the mask 109 and 200;
// 82 and 147 of 768 columns.)
// Rows of less than a piece end early.
template <typename T, int NV, int NW, bool WHOLE>
struct Cols {
  static constexpr int V = 16 / sizeof(T);
  using Row = Piece<T, V>[NV];
  // the first half of the pieces is there in every lane: narrower rows have fewer waves or pieces (waves_of)
  static constexpr int kFull = NV * V == 16 || NW > 1 ? NV / 2 : 0;
  int col[NV], left[NV], again[WHOLE ? 1 : NV];  // again: of the columns before it
  uint32_t mine[WHOLE ? 1 : NV - kFull][V];      // all ones where a column of these pieces is there and the lane's own, else 0
  __device__ __forceinline__ Cols(int wave, int lane, int d) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      col[j] = ((j * NW + wave % NW) * 64 + lane) * V;
      left[j] = d - col[j];
      if constexpr (!WHOLE) {
        again[j] = d >= V && left[j] > 0 && left[j] < V ? V - left[j] : 0;
        col[j] -= again[j];
        left[j] += again[j];
        if (j >= kFull) {
#pragma unroll
          for (int i = 0; i < V; ++i) mine[j - kFull][i] = in(j, i) ? ~0u : 0u;
        }
      }
    }
  }
  // whether a column is there, and whether it is the lane's own
  __device__ __forceinline__ bool has(int j, int i) const { return j < kFull || (WHOLE ? left[j] > 0 : i < left[j]); }
  __device__ __forceinline__ bool in(int j, int i) const { return has(j, i) && (WHOLE || i >= again[j]); }
  // A value as a row's sum takes it: zero where `in` is not. (Of a WHOLE row the caller's are zeros there, or it asks.)
  __device__ __forceinline__ float own(int j, int i, float v) const {
    if constexpr (WHOLE) return v;
    if (j < kFull) return v;
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & mine[j < kFull ? 0 : j - kFull][i]);
  }
  // a row's elements; zeros past it, and everywhere without a row
  __device__ __forceinline__ void load(Row& x, const void* base, int64_t at, bool have) const {
    const T* row = static_cast<const T*>(base) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j) x[j].template load<WHOLE>(row + col[j], have ? left[j] : 0);
  }
  __device__ __forceinline__ void store(void* base, int64_t at, const float (&v)[NV][V]) const {
    T* row = static_cast<T*>(base) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Piece<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = (T)v[j][i];
      o.template store<WHOLE>(row + col[j], left[j]);
    }
  }
  // a vector of weights as float32, `other` where there is none or past the row
  template <typename W>
  __device__ __forceinline__ void weights_of(float (&o)[NV][V], const W* w, float other) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Piece<W, V> p;
      p.template load<WHOLE>(w + col[j], left[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = has(j, i) ? (float)p.v[i] : other;
    }
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

template <typename T, int NV, int NW, bool POST, bool WHOLE>
__global__ void __launch_bounds__(kThreads) residual_norm_fwd_kernel(ResidualNormArgs a) {
  using C = Cols<T, NV, NW, WHOLE>;
  constexpr int V = C::V, NG = kWaves / NW;  // rows of a workgroup at a time
  __shared__ float red[2][2 * kWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const C c(wave, lane, a.d);
  const float inv = 1.0f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * NG;
  typename C::Row x, r, g, nx, nr, ng;
  int64_t row = (int64_t)blockIdx.x * NG + wave / NW;
  c.load(x, a.x, row * a.sx, row < a.M);
  c.load(r, a.r, row * a.sr, row < a.M);
  if (a.gate) c.load(g, a.gate, row * a.sg, row < a.M);
  float w[NV][V], b[NV][V], pw[NV][V], pb[NV][V], k[NV][V];
  c.weights(w, a.w, a.w32, 1.0f);
  c.weights(b, a.b, a.w32, 0.0f);
  c.weights(k, a.scale, a.w32, 1.0f);
  if constexpr (POST) {
    c.weights(pw, a.pw, a.w32, 1.0f);
    c.weights(pb, a.pb, a.w32, 0.0f);
  }
  int par = 0;
  auto sum = [&](float s) {
    float none = 0.0f;
    row_sum2<NW>(s, none, red[par], wave);
    par ^= 1;
    return s;
  };
  float h[NV][V];
  // mu and s of the values in h
  auto moments = [&](float& mu, float& rs) {
    mu = 0.0f;
    if (!a.rms) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) s += c.own(j, i, h[j][i]);
      mu = sum(s) * inv;
    }
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = c.own(j, i, h[j][i] - mu);
        sq += !WHOLE || c.has(j, i) ? e * e : 0.0f;
      }
    rs = 1.0f / sqrtf(sum(sq) * inv + a.eps);
  };
  // base, and so the number of barriers, is the same for all rows of the workgroup
  for (int64_t base = (int64_t)blockIdx.x * NG; base < a.M; base += step, row += step) {
    const bool more = row + step < a.M;
    c.load(nx, a.x, (row + step) * a.sx, more);
    c.load(nr, a.r, (row + step) * a.sr, more);
    if (a.gate) c.load(ng, a.gate, (row + step) * a.sg, more);
    float mu1 = 0.0f, rs1 = 1.0f, mu2, rs2;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) h[j][i] = (float)x[j].v[i];
    if constexpr (POST) {
      moments(mu1, rs1);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) h[j][i] = (h[j][i] - mu1) * rs1 * pw[j][i] + pb[j][i];
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = a.gate ? k[j][i] * (float)g[j].v[i] : k[j][i];
        h[j][i] = !WHOLE || c.has(j, i) ? a.alpha * (float)r[j].v[i] + q * h[j][i] : 0.0f;
      }
    moments(mu2, rs2);
    if (row < a.M) {
      c.store(a.h, row * a.d, h);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) h[j][i] = (h[j][i] - mu2) * rs2 * w[j][i] + b[j][i];
      c.store(a.y, row * a.d, h);
      if (a.stats && lane == 0 && wave % NW == 0)
        reinterpret_cast<f32x4_t*>(a.stats)[row] = f32x4_t{mu1, rs1, mu2, rs2};
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = nx[j];
      r[j] = nr[j];
      if (a.gate) g[j] = ng[j];
    }
  }
}

// Column sums in the order of the partial rows' slots.
enum Sum { kDw, kDb, kDscale, kDpw, kDpb, kSums };

template <typename T, int NV, int NW, bool POST, bool WHOLE>
__global__ void __launch_bounds__(kThreads) residual_norm_bwd_kernel(ResidualNormArgs a) {
  using C = Cols<T, NV, NW, WHOLE>;
  constexpr int V = C::V, NG = kWaves / NW;
  constexpr int S = POST ? kSums : kDscale + 1;
  // The workgroup's rows' sums meet in LDS: of each piece V rows of 64 lanes, 64 / V apart in banks, so that neither the lanes
  // that write a row nor the threads that read columns in order fall in the same ones. Two sums take turns.
  constexpr int P = 64 + 64 / V, PIECE = V * P, ROW = NV * NW * PIECE;
  __shared__ float red[2][2 * kWaves];
  __shared__ float fold[2][NG > 1 ? NG * ROW : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const C c(wave, lane, a.d);
  const float inv = 1.0f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * NG;
  float w[NV][V], pw[NV][V], pb[NV][V], k[NV][V], total[S][NV][V];
  c.weights(w, a.w, a.w32, 1.0f);
  c.weights(k, a.scale, a.w32, 1.0f);
  if constexpr (POST) {
    c.weights(pw, a.pw, a.w32, 1.0f);
    c.weights(pb, a.pb, a.w32, 0.0f);
  }
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) total[s][j][i] = 0.0f;
  struct Rows {
    typename C::Row x, r, g, dh, dy;
    f32x4_t st;
  };
  auto load = [&](Rows& o, int64_t at) __attribute__((always_inline)) {
    const bool have = at < a.M;
    c.load(o.x, a.x, at * a.sx, have);
    c.load(o.r, a.r, at * a.sr, have);
    if (a.gate) c.load(o.g, a.gate, at * a.sg, have);
    if (a.dh) c.load(o.dh, a.dh, at * a.sdh, have);
    if (a.dy) c.load(o.dy, a.dy, at * a.sdy, have);
    o.st = have ? reinterpret_cast<const f32x4_t*>(a.stats)[at] : f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  int64_t row = (int64_t)blockIdx.x * NG + wave / NW;
  int par = 0;
  auto sums = [&](const Rows& rows) __attribute__((always_inline)) {
    const auto &x = rows.x, &r = rows.r, &g = rows.g, &dh = rows.dh, &dy = rows.dy;
    const f32x4_t st = rows.st;
    const float mu1 = st[0], rs1 = st[1], mu2 = st[2], rs2 = st[3];
    const bool have = row < a.M;
    // Without a row all of these are zeros. Past a row's end dy, dh and what is added up are zeros, too, but for g, which
    // the row's means would enter: it is the one that is masked (of rows that are not WHOLE, what goes into sums is).
    float hh[NV][V], xh[NV][V], o[NV][V];  // hh: norm(h), then g; xh: norm(x), or x
    auto block = [&](int j, int i) { return POST ? xh[j][i] * pw[j][i] + pb[j][i] : xh[j][i]; };  // t
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = (float)x[j].v[i];
        if constexpr (POST) xh[j][i] = (xh[j][i] - mu1) * rs1;
        const float q = a.gate ? k[j][i] * (float)g[j].v[i] : k[j][i];
        const float n = (a.alpha * (float)r[j].v[i] + q * block(j, i) - mu2) * rs2;
        hh[j][i] = n;
        if (a.dy) {
          const float d = (float)dy[j].v[i], wdy = c.own(j, i, d * w[j][i]);
          s1 += wdy;
          s2 += wdy * c.own(j, i, n);
          total[kDw][j][i] += d * n;
          total[kDb][j][i] += d;
        }
      }
    if (a.dy) {
      row_sum2<NW>(s1, s2, red[par], wave);
      par ^= 1;
    }
    const float c1 = a.rms ? 0.0f : s1 * inv, c2 = s2 * inv;
    s1 = s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float e = a.dh ? (float)dh[j].v[i] : 0.0f;
        if (a.dy) e += rs2 * ((float)dy[j].v[i] * w[j][i] - c1 - hh[j][i] * c2);
        e = !WHOLE || c.has(j, i) ? e : 0.0f;
        hh[j][i] = e;
        const float f = a.gate ? e * (float)g[j].v[i] : e, q = f * k[j][i];
        total[kDscale][j][i] += f * block(j, i);
        if constexpr (POST) {
          total[kDpw][j][i] += q * xh[j][i];
          total[kDpb][j][i] += q;
          o[j][i] = q * pw[j][i];
          const float p = c.own(j, i, o[j][i]);
          s1 += p;
          s2 += p * c.own(j, i, xh[j][i]);
        } else {
          o[j][i] = q;
        }
      }
    if (POST && a.dx) {
      row_sum2<NW>(s1, s2, red[par], wave);
      par ^= 1;
      const float e1 = a.rms ? 0.0f : s1 * inv, e2 = s2 * inv;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) o[j][i] = rs1 * (o[j][i] - e1 - xh[j][i] * e2);
    }
    if (have) {
      if (a.dx) c.store(a.dx, row * a.d, o);
      if (a.dgate) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) o[j][i] = hh[j][i] * k[j][i] * block(j, i);
        c.store(a.dgate, row * a.d, o);
      }
      if (a.dr) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) o[j][i] = a.alpha * hh[j][i];
        c.store(a.dr, row * a.d, o);
      }
    }
  };
  // Rows are loaded while others are summed: two ahead in three sets of registers, one ahead where a lane has 16 elements.
  // (The sets take turns by name: handing registers on would wait for their loads.)
  int64_t base = (int64_t)blockIdx.x * NG;
  if constexpr (NV == 1) {
    Rows r0, r1, r2;
    load(r0, row);
    load(r1, row + step);
    auto turn = [&](Rows& now, Rows& next) __attribute__((always_inline)) {
      load(next, row + 2 * step);
      sums(now);
      base += step;
      row += step;
      return base < a.M;  // the same for all rows of the workgroup, and so is the number of barriers
    };
    while (turn(r0, r2) && turn(r1, r0) && turn(r2, r1)) {
    }
  } else {
    Rows r0, r1;
    load(r0, row);
    auto turn = [&](Rows& now, Rows& next) __attribute__((always_inline)) {
      load(next, row + step);
      sums(now);
      base += step;
      row += step;
      return base < a.M;
    };
    while (turn(r0, r1) && turn(r1, r0)) {
    }
  }
  if (!a.part) return;
  // wanted sums one behind the other, [parts][wanted][d]
  float* part = a.part + (int64_t)blockIdx.x * a.wanted * a.d;
  int turn = 0;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (!a.sums[s]) continue;
    if constexpr (NG > 1) {
      float* f = fold[turn & 1];
      ++turn;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
          f[wave / NW * ROW + (j * NW + wave % NW) * PIECE + i * P + lane] = total[s][j][i];
      __syncthreads();
      for (int k = threadIdx.x; k < a.d; k += kThreads) {
        const int piece = k / V, left = a.d - piece * V;
        const int i = k % V + (!WHOLE && a.d >= V && left < V ? V - left : 0);  // in the lane that has it as its own
        const float* at = f + piece / 64 * PIECE + i * P + piece % 64;
        float t = at[0];
#pragma unroll
        for (int q = 1; q < NG; ++q) t += at[q * ROW];
        part[k] = t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c.in(j, i)) part[c.col[j] + i] = total[s][j][i];
    }
    part += a.d;
  }
}

// The wanted sums: the columns of `parts` rows, 16 a workgroup, its threads 64 rows at a time.
template <typename O>
__global__ void __launch_bounds__(1024) residual_norm_join_kernel(ResidualNormArgs a, int parts) {
  __shared__ float sums[64][17];
  const int c = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int64_t n = (int64_t)a.wanted * a.d, at = (int64_t)blockIdx.x * 16 + c;
  float s = 0.0f;
  if (at < n) {
#pragma unroll 4
    for (int p = group; p < parts; p += 64) s += a.part[p * n + at];
  }
  sums[group][c] = s;
  __syncthreads();
#pragma unroll
  for (int half = 32; half >= 4; half /= 2) {  // to four sums a column
    if (group < half) sums[group][c] += sums[group + half][c];
    __syncthreads();
  }
  if (group == 0 && at < n) {
    s = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
    int slot = (int)(at / a.d);
    const int k = (int)(at - (int64_t)slot * a.d);
    for (int q = 0; q < kSums; ++q) {
      if (!a.sums[q]) continue;
      if (slot-- == 0) static_cast<O*>(a.sums[q])[k] = (O)s;
    }
  }
}

// Workgroups for M rows, `group` at a time: as many as run at once (per_cu on each compute unit).
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

// Waves of a row, with 16 elements a lane in the forward and 8 in the backward (16 in the widest rows).
int waves_of(int d, bool bwd) {
  int nw = 1;
  while (nw < kWaves && d > 64 * nw * (bwd ? 8 : 16)) nw *= 2;
  return nw;
}

template <typename T, int E, int NW, bool POST, bool WHOLE, bool BWD>
int run(const ResidualNormArgs& a, hipStream_t s) {
  constexpr int NV = E * (int)sizeof(T) / 16;
  if constexpr (BWD) {
    static const int n = held(reinterpret_cast<const void*>(residual_norm_bwd_kernel<T, NV, NW, POST, WHOLE>));
    const int grid = grid_of(a.M, kWaves / NW, n < kBwdPerCu ? n : kBwdPerCu);
    residual_norm_bwd_kernel<T, NV, NW, POST, WHOLE><<<grid, kThreads, 0, s>>>(a);
    return grid;
  } else {
    static const int n = held(reinterpret_cast<const void*>(residual_norm_fwd_kernel<T, NV, NW, POST, WHOLE>));
    const int grid = grid_of(a.M, kWaves / NW, n);
    residual_norm_fwd_kernel<T, NV, NW, POST, WHOLE><<<grid, kThreads, 0, s>>>(a);
    return grid;
  }
}

template <typename T, bool POST, bool WHOLE>
int run_row(const ResidualNormArgs& a, bool bwd, hipStream_t s) {
  const int nw = waves_of(a.d, bwd);
  const bool eight = a.d <= 64 * nw * 8;
  if (bwd) {
    switch (nw) {
      case 1: return run<T, 8, 1, POST, WHOLE, true>(a, s);
      case 2: return run<T, 8, 2, POST, WHOLE, true>(a, s);
      case 4: return run<T, 8, 4, POST, WHOLE, true>(a, s);
      default: return eight ? run<T, 8, 8, POST, WHOLE, true>(a, s) : run<T, 16, 8, POST, WHOLE, true>(a, s);
    }
  }
  switch (nw) {
    case 1: return eight ? run<T, 8, 1, POST, WHOLE, false>(a, s) : run<T, 16, 1, POST, WHOLE, false>(a, s);
    case 2: return run<T, 16, 2, POST, WHOLE, false>(a, s);
    case 4: return run<T, 16, 4, POST, WHOLE, false>(a, s);
    default: return run<T, 16, 8, POST, WHOLE, false>(a, s);
  }
}

template <typename T>
int launch(const ResidualNormArgs& a, bool bwd, hipStream_t s) {
  const bool whole = a.d % (16 / sizeof(T)) == 0;
  if (a.post) return whole ? run_row<T, true, true>(a, bwd, s) : run_row<T, true, false>(a, bwd, s);
  return whole ? run_row<T, false, true>(a, bwd, s) : run_row<T, false, false>(a, bwd, s);
}

int launch_kind(int kind, const ResidualNormArgs& a, bool bwd, hipStream_t s) {
  if (kind == FMX_DTYPE_F32) return launch<float>(a, bwd, s);
  if (kind == FMX_DTYPE_BF16) return launch<__bf16>(a, bwd, s);
  return launch<_Float16>(a, bwd, s);
}

}  // namespace

int residual_norm_parts(int64_t M, int d) { return grid_of(M, kWaves / waves_of(d, true), kBwdPerCu); }

hipError_t launch_residual_norm_fwd(int kind, const ResidualNormArgs& a, hipStream_t s) {
  launch_kind(kind, a, false, s);
  return hipGetLastError();
}

hipError_t launch_residual_norm_bwd(int kind, const ResidualNormArgs& a, hipStream_t s) {
  int parts = 0;  // no rows: the sums of nothing
  if (a.M > 0) {
    parts = launch_kind(kind, a, true, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.wanted) return hipSuccess;
  const unsigned grid = (unsigned)(((int64_t)a.wanted * a.d + 15) / 16);
  if (a.w32 || kind == FMX_DTYPE_F32)
    residual_norm_join_kernel<float><<<grid, 1024, 0, s>>>(a, parts);
  else if (kind == FMX_DTYPE_BF16)
    residual_norm_join_kernel<__bf16><<<grid, 1024, 0, s>>>(a, parts);
  else
    residual_norm_join_kernel<_Float16><<<grid, 1024, 0, s>>>(a, parts);
  return hipGetLastError();
}

}  // namespace fmx
