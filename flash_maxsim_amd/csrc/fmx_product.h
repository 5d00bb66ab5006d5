// What the tile products of the trained layers share (linear, gated linear, the
// optimizer's iteration): operands of 16 bits from memory to LDS and from there
// to MFMA's registers, the order of a stage's instructions, activations, and 8
// neighbouring outputs of a lane to and from memory.
//
// An operand stored [i, k] ("K-major") is read from LDS with 16-byte reads of 8
// k values; one stored [k, i] ("row-major") with transposing reads
// (ds_read_b64_tr_b16: of the 16 lanes that read a 4 x 16 block, lane l gets
// column l), so no operand is transposed in memory first. Stages of BK k values
// stream global -> LDS by DMA (16 bytes a lane) into NS buffers, the next stage
// in flight while one is multiplied. Chunk positions in LDS are XOR-swizzled so
// that the lanes of a read fall in distinct banks.
#pragma once

#include <type_traits>

#include "fmx_device.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf) {
  if (bf) {
    const __bf16 x = (__bf16)a, y = (__bf16)b;
    return (uint32_t)__builtin_bit_cast(uint16_t, x) | ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
  }
  const _Float16 x = (_Float16)a, y = (_Float16)b;
  return (uint32_t)__builtin_bit_cast(uint16_t, x) | ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
}
__device__ __forceinline__ float unpack(uint32_t bits16, bool bf) {
  return bf ? bf16_bits_to_float(bits16) : half_bits_to_float(bits16);
}

// ---- activations ----

// Phi(z), the normal distribution function, and e = exp(-z^2 / 2): Abramowitz and
// Stegun 7.1.26 (erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x), off
// by 1.5e-7 at most) at x = |z| / sqrt 2; the lower tail has no cancellation.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float a = __builtin_fabsf(z);
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752044f);  // exp(-z^2 / 2)
  const float t = __builtin_amdgcn_rcpf(fmaf(0.2316418882f, a, 1.0f));  // p / sqrt 2
  float q = fmaf(t, 0.5307027145f, -0.7265760135f);  // the halves of a5 .. a1
  q = fmaf(t, q, 0.7107068705f);
  q = fmaf(t, q, -0.142248368f);
  q = fmaf(t, q, 0.1274147960f);
  q = q * t * e;
  return z < 0.0f ? q : 1.0f - q;
}
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504089f));
}

// act(z), and with SLOPE act'(z). As a factor of a tail that is zero z is kept finite: their product would be NaN.
template <bool SLOPE>
__device__ __forceinline__ float act_value(float z, int act, float& slope) {
  const float f = SLOPE ? __builtin_fminf(__builtin_fmaxf(z, -1e4f), 1e4f) : z;
  switch (act) {
    case FMX_ACT_RELU:
      slope = z > 0.0f ? 1.0f : 0.0f;
      return z > 0.0f ? z : z != z ? z : 0.0f;
    case FMX_ACT_GELU: {
      float e;
      const float p = normal_cdf(z, e);
      slope = fmaf(f * 0.3989422804f, e, p);
      return z * p;
    }
    // z (1 + tanh u) / 2 = z sigmoid(2 u)
    case FMX_ACT_GELU_TANH: {
      const float s = sigmoid(1.5957691216f * z * fmaf(0.044715f, z * z, 1.0f));
      slope = s + f * s * (1.0f - s) * 1.5957691216f * fmaf(0.134145f, f * f, 1.0f);
      return z * s;
    }
    case FMX_ACT_SILU: {
      const float s = sigmoid(z);
      slope = s + f * s * (1.0f - s);
      return z * s;
    }
    default:
      slope = 1.0f;
      return z;
  }
}

// ---- epilogue: 8 consecutive outputs j .. j + 7 of row i, of which `left` exist ----

__device__ __forceinline__ u32x4_t pack8(const float (&v)[8], bool bf) {
  return u32x4_t{pack2(v[0], v[1], bf), pack2(v[2], v[3], bf), pack2(v[4], v[5], bf), pack2(v[6], v[7], bf)};
}

// Rows may begin at any element (odd widths): the 16-byte accesses need no more than 2-byte alignment here (gfx950
// under the HSA runtime takes them as they come; 1003 x 77 with 2-byte ones: dz 10 us, the forward 7.6; so 6 and 6.1).
__device__ __forceinline__ void store_raw(void* base, int64_t at, int left, const u32x4_t& w) {
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (left >= 8) {
    __builtin_memcpy(p, &w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = w[i / 2];
      if (i < left) p[i] = (uint16_t)((i & 1) ? x >> 16 : x);
    }
  }
}
__device__ __forceinline__ void store16(void* base, int64_t at, int left, const float (&v)[8], bool bf) {
  store_raw(base, at, left, pack8(v, bf));
}

__device__ __forceinline__ u32x4_t load_raw(const void* base, int64_t at, int left) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (left >= 8) {
    __builtin_memcpy(&v, p, 16);
    return v;
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  // the last one again in place of those past it (left >= 1): no branches, all loads in flight
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = p[i < left ? i : left - 1];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i / 2] |= (i < left ? e[i] : 0u) << (16 * (i & 1));
  return u32x4_t{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ void unpack8(float (&v)[8], const u32x4_t& w, bool bf) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = w[i / 2];
    v[i] = unpack((i & 1) ? x >> 16 : x & 0xffffu, bf);
  }
}
__device__ __forceinline__ void load16(float (&v)[8], const void* base, int64_t at, int left, bool bf) {
  unpack8(v, load_raw(base, at, left), bf);
}

// What follows the sums: a form's own activation (FMX_ACT_*: the forward's tile kernels are compiled for each, their
// unrolled epilogues hold the code many times over), one named at run time, or nothing (dx, dw).
constexpr int kAnyAct = -1, kNoEpilogue = -2;

template <int ACT, bool SLOPE>
__device__ __forceinline__ void activate(float (&v)[8], float (&slope)[8], int act) {
  if constexpr (ACT >= 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = act_value<SLOPE>(v[k], ACT, slope[k]);
  } else {
    switch (act) {  // uniform: one test for the eight
#define FMX_CASE(A) \
  case A: activate<A, SLOPE>(v, slope, A); break
      FMX_CASE(FMX_ACT_RELU);
      FMX_CASE(FMX_ACT_GELU);
      FMX_CASE(FMX_ACT_GELU_TANH);
      FMX_CASE(FMX_ACT_SILU);
#undef FMX_CASE
      default: break;
    }
  }
}

// ---- the product ----

constexpr int BK = 64;  // k values of a stage: 128-byte rows of a K-major operand, whole lines of memory

// One operand's side of a tile: T rows (of i or j), from row r0 on.
template <bool MAJ, bool PAIR, int T, int NT>
struct Side {
  static constexpr int kChunks = T * BK / 8;            // 16-byte chunks of a stage
  static constexpr int kLoads = kChunks / NT;           // of a thread
  static constexpr int kRow = MAJ ? T / 8 : BK / 8;     // chunks of an LDS row
  static_assert(kChunks % NT == 0 && (MAJ || NT % (8 * kRow) == 0), "a stage splits evenly over the threads");
  const char* base;
  int64_t step;        // bytes from one stage to the next
  uint32_t off[kLoads];
  int kfirst;          // the first chunk's (first) k inside its stage

  // position of chunk ch of LDS row r is ch ^ key(r)
  static __device__ __forceinline__ int key(int r) {
    if constexpr (MAJ) return (2 * (r & 3) | (kRow > 8 ? ((r >> 3) & 1) << 3 : 0)) & (kRow - 1);
    // PAIR: the rows of one fragment are 0-3, 8-11, 16-19, 24-27 (and 4 more)
    return PAIR ? (r & 3) | ((r >> 3) & 1) << 2 : r & 7;
  }

  __device__ __forceinline__ Side(const void* p, int64_t stride, int64_t r0, int64_t rows, int64_t k0, int tid) {
    base = static_cast<const char*>(p) + (MAJ ? k0 * stride + r0 : r0 * stride + k0) * 2;
    step = (MAJ ? stride : 1) * (int64_t)BK * 2;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int at = n * NT + tid, r = at / kRow, ch = (at % kRow) ^ key(r);
      if (n == 0) kfirst = MAJ ? r : ch * 8;
      const int row = MAJ ? ch * 8 : r;  // of i or j, inside the tile
      off[n] = r0 + row < rows ? (uint32_t)(r * stride * 2 + ch * 16) : kOOB;
    }
  }
  // Stage `it` to LDS; kleft: k values left from its start (those at or past it read as zeros).
  // K-major: a thread's chunks lie 8 rows (or a multiple) apart, so they hold the same k.
  __device__ __forceinline__ void issue(unsigned char* lds, int it, int kleft, int wave) const {
    issue_from(base + it * step, lds, kleft, wave);
  }
  // The same from another matrix of the same stride; `from`: the stage's first element.
  __device__ __forceinline__ void issue_from(const char* from, unsigned char* lds, int kleft, int wave) const {
    const rsrc_t r = make_rsrc(from, 0x7fffffffu);
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      dma16_lds<false>(r, lds + (n * NT + wave * 64) * 16, kfirst + (MAJ ? n * (NT / kRow) : 0) < kleft ? off[n] : kOOB);
  }
};

// Fragment reader of one operand: 16 rows x 32 k of fragment f, k-step kk.
template <bool MAJ, bool PAIR, int T>
struct Frags {
  uint32_t at[MAJ ? 1 : BK / 32];
  __device__ __forceinline__ Frags(int row0, int lane) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (MAJ) {
      const int q = c >> 2, s = c & 3, r = 8 * g + q;
      at[0] = (uint32_t)(r * T * 2 + (((row0 >> 3) + (s >> 1)) ^ Side<MAJ, PAIR, T, 64 * 8>::key(r)) * 16 + 8 * (s & 1));
    } else {
      const int row = row0 + (PAIR ? 8 * (c >> 2) + (c & 3) : c);
      const int key = c & 7;  // of the row, and of all others of the lane's fragments
#pragma unroll
      for (int kk = 0; kk < BK / 32; ++kk) at[kk] = (uint32_t)(row * BK * 2 + ((kk * 4 + g) ^ key) * 16);
    }
  }
  __device__ __forceinline__ u32x4_t read(const unsigned char* lds, int f, int kk) const {
    if constexpr (MAJ) {
      typedef __attribute__((address_space(3))) s16x4_t lds_t;
      // chunk 2 f further: row0 is a multiple of 8 chunks and rows are powers of two apart, so it is an
      // exclusive or of the address; k rows 32 kk + 8 g + 0..3, then + 4..7 (the key of row r + 4 is that of r)
      const unsigned char* p = lds + (at[0] ^ (uint32_t)(32 * f));
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(p + (32 * kk) * T * 2));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(p + (32 * kk + 4) * T * 2));
      const u32x2_t l = __builtin_bit_cast(u32x2_t, lo), h = __builtin_bit_cast(u32x2_t, hi);
      return u32x4_t{l[0], l[1], h[0], h[1]};
    } else {
      const int o = PAIR ? (f >> 1) * 32 + 4 * (f & 1) : f * 16;
      return *reinterpret_cast<const u32x4_t*>(lds + at[kk] + o * BK * 2);
    }
  }
};

// Which tile of ti x tj, and which part of k, a workgroup computes. Workgroups go to the eight XCDs in turn; each XCD
// takes a run of consecutive tiles, which share operand rows in its L2. Runs of `band` tile rows are walked column by
// column. (32-bit divisions: a launch has fewer than 2^32 threads.)
struct Place {
  uint32_t split, row, col;
  __device__ __forceinline__ Place(uint32_t id, uint32_t ti, uint32_t tj, uint32_t splits, uint32_t bands) {
    const uint32_t tiles = ti * tj, total = tiles * splits, per = total / 8, x = id & 7, rest = total & 7;
    id = (id >> 3) + x * per + (x < rest ? x : rest);
    split = splits > 1 ? id / tiles : 0;
    uint32_t t = id - split * tiles;
    const uint32_t band = t / (bands * tj);
    const uint32_t rows = ti - band * bands < bands ? ti - band * bands : bands;
    t -= band * bands * tj;
    col = t / rows;
    row = band * bands + (t - col * rows);
  }
};

// LDS buffers are separate objects, named at compile time in the unrolled stage
// loop: the compiler then knows that reads of one do not alias the DMA writes in
// flight to another and puts no wait for those in front of them.
__device__ __forceinline__ void stage_barrier() {
  __asm__ volatile("" ::: "memory");
  wait_lds();
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}

// The stages of a product, `nit` of them. The caller's lambdas: buffer(s) is LDS buffer s % NS; issue(lds, it) starts
// the LOADS DMAs of stage `it`; read(set, lds, kk) reads the READS fragments of k-step kk into a set of registers;
// multiply(set) issues its MFMAS; besides(set) may multiply more with them.
//
// Fragments of one k-step of 32: a set is multiplied while the next one is read. Before the first read of a new
// stage every wave waits for its own DMA of it and for its reads of the old one, then all meet; the
// old one's buffer takes the DMA of the stage NS ahead.
constexpr std::integral_constant<int, 0> set0{};
constexpr std::integral_constant<int, 1> set1{};

template <int NS, int LOADS, int READS, int MFMAS, class Buffer, class Issue, class Read, class Multiply, class Besides>
__device__ __forceinline__ void run_stages(int nit, const Buffer& buffer, const Issue& issue, const Read& read,
                                           const Multiply& multiply, const Besides& besides) {
  static_assert(NS == 2 || NS == 4, "stage buffers");
  // The order of the instructions after a barrier: the multiplication of the set at hand runs from the
  // first one on, between the loads and reads.
  auto interleave = [&]() __attribute__((always_inline)) {
    constexpr int R = READS > 12 ? 2 : 1;
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
#pragma unroll
    for (int n = 0; n < READS / R; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);
  };
  auto stage = [&](auto s, int it) __attribute__((always_inline)) {
    read(set1, buffer(s), 1);
    multiply(set0);
    besides(set0);
    wait_vmem<(NS - 2) * LOADS>();
    stage_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue(buffer(s), it + NS);
    read(set0, buffer(std::integral_constant<int, decltype(s)::value + 1>{}), 0);
    multiply(set1);
    interleave();
    __builtin_amdgcn_sched_barrier(0);
    besides(set1);
  };
  constexpr std::integral_constant<int, 2> two{};
  constexpr std::integral_constant<int, 3> three{};
  issue(buffer(set0), 0);
  issue(buffer(set1), 1);
  if constexpr (NS > 2) {
    issue(buffer(two), 2);
    issue(buffer(three), 3);
  }
  wait_vmem<(NS - 1) * LOADS>();
  stage_barrier();
  read(set0, buffer(set0), 0);
  for (int it = 0; it < nit; it += NS) {
    stage(set0, it);
    if (it + 1 < nit) stage(set1, it + 1);
    if constexpr (NS > 2) {
      if (it + 2 < nit) stage(two, it + 2);
      if (it + 3 < nit) stage(three, it + 3);
    }
  }
  wait_vmem<0>();  // the stages past the end: their (empty) DMA writes no longer reach LDS after this wave ends
}

}  // namespace
}  // namespace fmx
