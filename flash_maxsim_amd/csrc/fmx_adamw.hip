// AdamW (decoupled weight decay) over many tensors in one launch, with the two
// moments held in float32 or in 8 bits.
//
//   g = grad * grad_scale
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Every product and sum is rounded to float32 by itself (no contraction into
// fma), so a new 8-bit code never depends on how the compiler fused the
// formula; the root is the device library's sqrtf. The parameter is rounded to
// its own type once, at the end.
//
// 8-bit moments: blocks of 256 elements of one tensor share a float32 scale q.
// The first moment is c |c| q with c an int8 code, q = max |m| / 127^2; of the
// second the root is held, c^2 q with c a uint8 code, q = max sqrt(v) / 255^2:
// a quadratic grid, whose steps are 1.6 % (0.8 %) of the largest value at the
// top and shrink towards zero, where most values of a block lie. A code is the
// number of grid midpoints (c - 1/2)^2 at or below |m| / q: y = |m| (127^2 / max)
// is compared with c^2 + c + 1/4, which float32 holds exactly. A root that is
// not zero keeps at least code 1, so no element's step grows because its second
// moment was rounded to nothing. A block with a value that is not finite
// decodes to NaN: of the first moment zeros times an infinite scale, of the
// second, whose codes of at least 1 would make that infinite (steps of zero for
// all of the block from then on), by a scale that is NaN.
//
// Bound by HBM: 28 bytes a parameter in float32, 10 with bf16 parameters and
// 8-bit moments, against about 40 (80) vector operations.
#include "fmx_device.h"
#include "fmx_layers.h"

#include "../../include/fmx.h"

#pragma clang fp contract(off)

namespace fmx {
namespace {

constexpr int kThreads = 256;
constexpr int kElems = 8;                         // per lane: 32 lanes hold a block of 256
constexpr int kChunk = kThreads * kElems;         // elements a workgroup takes
constexpr int kMaxTensors = 76;                   // of one launch: the table travels in the kernel's arguments
constexpr float kTinyBlock = 0x1p-110f;           // a block below this is held as zeros (127^2 / it overflows soon after)

// A tensor in 48 bytes (user-space addresses have 48 bits), so that 4 KB of arguments hold 76 of them: every launch
// fills the GPU and drains it again, about 5 us that 150 tensors paid four times with 64 bytes each.
struct Entry {
  uint32_t lo[7];   // low halves of param, grad, m, v, ms, vs, copy
  uint32_t hi[4];   // their bits 32 .. 47 in pairs; the last one's pair: all arrays allow 16-byte (codes: 8-byte) accesses
  uint32_t n;
};
struct Table {
  Entry t[kMaxTensors];
  int32_t first[kMaxTensors + 1];                 // first workgroup of each tensor
  int32_t count;
};
static_assert(sizeof(Table) + sizeof(AdamWScalars) <= 4096, "kernel arguments");

__device__ __forceinline__ void* address(const Entry& e, int k) {
  const uint32_t hi = (k & 1) ? e.hi[k / 2] >> 16 : e.hi[k / 2] & 0xffffu;
  return reinterpret_cast<void*>((uint64_t)hi << 32 | e.lo[k]);
}

template <typename T, int V>
struct __attribute__((aligned(sizeof(T) * V >= 16 ? 16 : sizeof(T) * V))) Pack {
  T v[V];
};

// Elements i0 .. i0 + 7 of an array of n; unless WHOLE those at or past n read as zero and are not written.
template <bool WHOLE, typename T, typename F>
__device__ __forceinline__ void load8(const T* p, int64_t i0, int64_t n, F&& put) {
  if constexpr (WHOLE) {
    const Pack<T, kElems> x = *reinterpret_cast<const Pack<T, kElems>*>(p + i0);
#pragma unroll
    for (int i = 0; i < kElems; ++i) put(i, x.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kElems; ++i) put(i, i0 + i < n ? p[i0 + i] : T(0));
  }
}
template <bool WHOLE, typename T, typename F>
__device__ __forceinline__ void store8(T* p, int64_t i0, int64_t n, F&& get) {
  if constexpr (WHOLE) {
    Pack<T, kElems> x;
#pragma unroll
    for (int i = 0; i < kElems; ++i) x.v[i] = get(i);
    *reinterpret_cast<Pack<T, kElems>*>(p + i0) = x;
  } else {
#pragma unroll
    for (int i = 0; i < kElems; ++i)
      if (i0 + i < n) p[i0 + i] = get(i);
  }
}

// Largest value over the 32 lanes of each half of the wave, NaN if any is.
__device__ __forceinline__ float half_max(float v) {
  v = vmax(v, dpp_mov<0xB1>(v));
  v = vmax(v, dpp_mov<0x4E>(v));
  v = vmax(v, dpp_mov<0x141>(v));
  v = vmax(v, dpp_mov<0x140>(v));
  float lo, hi;
  halves16(v, lo, hi);
  return vmax(lo, hi);
}

// The code of y = |value| top^2 / max: see above. v_sqrt_f32 is within an ulp of
// the root, so a candidate from a root two ulps or more too small is the code or
// one below it, and one comparison settles it (c^2 + c + 1/4 has 18 bits at most). y
// is at most a rounding above top^2, so the code is at most top; not a number: 0.
__device__ __forceinline__ int code_of(float y) {
  const float c = rintf(__builtin_amdgcn_sqrtf(y) * 0x1.fffff8p-1f);
  return (int)c + (y >= fmaf(c, c, c + 0.25f) ? 1 : 0);
}

template <typename P, typename G, typename C, int BITS, bool WHOLE>
__device__ __forceinline__ void adamw_chunk(const AdamWTensor& t, const AdamWScalars& sc, int64_t i0) {
  const int64_t n = t.n;
  float p[kElems], g[kElems], m[kElems], r[kElems];
  load8<WHOLE>(static_cast<const P*>(t.param), i0, n, [&](int i, P x) { p[i] = (float)x; });
  load8<WHOLE>(static_cast<const G*>(t.grad), i0, n, [&](int i, G x) { g[i] = (float)x; });
  const int64_t block = i0 / 256;
  if constexpr (BITS == 8) {
    const bool in = WHOLE || i0 < n;
    const float qm = in ? t.ms[block] : 0.0f, qv = in ? t.vs[block] : 0.0f;
    load8<WHOLE>(static_cast<const int8_t*>(t.m), i0, n, [&](int i, int8_t c) {
      const float f = (float)c;
      m[i] = (f * __builtin_fabsf(f)) * qm;
    });
    load8<WHOLE>(static_cast<const uint8_t*>(t.v), i0, n, [&](int i, uint8_t c) {
      const float f = (float)c;
      const float root = (f * f) * qv;
      r[i] = root * root;
    });
  } else {
    load8<WHOLE>(static_cast<const float*>(t.m), i0, n, [&](int i, float x) { m[i] = x; });
    load8<WHOLE>(static_cast<const float*>(t.v), i0, n, [&](int i, float x) { r[i] = x; });
  }
  const float scale = sc.grad_scale ? *sc.grad_scale : 1.0f;
  float v[kElems];
#pragma unroll
  for (int i = 0; i < kElems; ++i) {
    const float gi = g[i] * scale;
    m[i] = m[i] * sc.beta1 + gi * sc.omb1;
    v[i] = r[i] * sc.beta2 + (gi * gi) * sc.omb2;
    r[i] = sqrtf(v[i]);
    // m over the denominator by the hardware's reciprocal (one ulp): of the step,
    // not of the state
    const float step = m[i] * __builtin_amdgcn_rcpf(r[i] * sc.root + sc.eps);
    p[i] = p[i] * sc.keep - step * sc.rate;
  }
  store8<WHOLE>(static_cast<P*>(t.param), i0, n, [&](int i) { return (P)p[i]; });
  if (t.copy) store8<WHOLE>(static_cast<C*>(t.copy), i0, n, [&](int i) { return (C)p[i]; });
  if constexpr (BITS == 8) {
    // elements past the end: their moments are zero, as all they were made of
    float bm = 0.0f, bv = 0.0f;
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
      bm = vmax(bm, __builtin_fabsf(m[i]));
      bv = vmax(bv, r[i]);
    }
    bm = half_max(bm);
    bv = half_max(bv);
    const bool zm = bm < kTinyBlock, zv = bv < kTinyBlock;
    const float im = zm ? 0.0f : 16129.0f / bm, iv = zv ? 0.0f : 65025.0f / bv;
    if ((threadIdx.x & 31) == 0 && (WHOLE || i0 < n)) {
      t.ms[block] = zm ? 0.0f : bm / 16129.0f;
      t.vs[block] = zv ? 0.0f : bv < __builtin_inff() ? bv / 65025.0f : __builtin_nanf("");
    }
    store8<WHOLE>(static_cast<int8_t*>(t.m), i0, n, [&](int i) {
      const int c = code_of(__builtin_fabsf(m[i]) * im);
      return (int8_t)(m[i] < 0.0f ? -c : c);
    });
    const float least = zv ? __builtin_inff() : 0.0f;  // roots above it keep code 1
    store8<WHOLE>(static_cast<uint8_t*>(t.v), i0, n, [&](int i) {
      const int c = code_of(r[i] * iv), one = r[i] > least ? 1 : 0;
      return (uint8_t)(c > one ? c : one);
    });
  } else {
    store8<WHOLE>(static_cast<float*>(t.m), i0, n, [&](int i) { return m[i]; });
    store8<WHOLE>(static_cast<float*>(t.v), i0, n, [&](int i) { return v[i]; });
  }
}

// The waves whose 512 elements are all there and aligned take the loads as they come, one branch for all of
// them (a test at each array made every load wait for the one before: 198 us for 64 M bf16 parameters with
// 8-bit moments, 168 so).
template <typename P, typename G, typename C, int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(Table tab, AdamWScalars sc) {
  // the tensor whose workgroups include this one
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int)blockIdx.x >= tab.first[mid])
      lo = mid;
    else
      hi = mid;
  }
  const Entry e = tab.t[lo];
  const AdamWTensor t = {address(e, 0),
                         address(e, 1),
                         address(e, 2),
                         address(e, 3),
                         static_cast<float*>(address(e, 4)),
                         static_cast<float*>(address(e, 5)),
                         address(e, 6),
                         (int64_t)e.n};
  const int64_t start = (int64_t)((int)blockIdx.x - tab.first[lo]) * kChunk;
  const int64_t end = start + (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + 1) * (64 * kElems);
  const int64_t i0 = start + threadIdx.x * kElems;
  if ((e.hi[3] >> 16) && end <= t.n)
    adamw_chunk<P, G, C, BITS, true>(t, sc, i0);
  else if (end - 64 * kElems < t.n)  // whole waves: the lanes of a block meet in its largest values
    adamw_chunk<P, G, C, BITS, false>(t, sc, i0);
}

// The values of 8-bit codes: c |c| q, and for the second moment its square. One
// lane takes eight; 10 bytes an element move.
template <bool SECOND>
__global__ void __launch_bounds__(kThreads) adamw_decode_kernel(const void* codes, const float* scales, int64_t n,
                                                                float* out, int vec) {
  using C = std::conditional_t<SECOND, uint8_t, int8_t>;
  const int64_t i0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kElems;
  if (i0 >= n) return;
  const float q = scales[i0 / 256];
  float x[kElems];
  auto put = [&](int i, C c) {
    const float f = (float)c;
    const float e = (f * __builtin_fabsf(f)) * q;
    x[i] = SECOND ? e * e : e;
  };
  auto get = [&](int i) { return x[i]; };
  if (vec && i0 + kElems <= n) {
    load8<true>(static_cast<const C*>(codes), i0, n, put);
    store8<true>(out, i0, n, get);
  } else {
    load8<false>(static_cast<const C*>(codes), i0, n, put);
    store8<false>(out, i0, n, get);
  }
}

template <typename P, typename G, typename C>
hipError_t launch_bits(int bits, int grid, const Table& tab, const AdamWScalars& sc, hipStream_t s) {
  if (bits == 8)
    adamw_kernel<P, G, C, 8><<<grid, kThreads, 0, s>>>(tab, sc);
  else
    adamw_kernel<P, G, C, 32><<<grid, kThreads, 0, s>>>(tab, sc);
  return hipGetLastError();
}

hipError_t launch_types(int pkind, int gkind, int ckind, int bits, int grid, const Table& tab, const AdamWScalars& sc,
                        hipStream_t s) {
  // gradients in the parameters' type or in float32; only float32 parameters have copies
  if (pkind == FMX_DTYPE_F16)
    return gkind == FMX_DTYPE_F32 ? launch_bits<_Float16, float, _Float16>(bits, grid, tab, sc, s)
                                  : launch_bits<_Float16, _Float16, _Float16>(bits, grid, tab, sc, s);
  if (pkind == FMX_DTYPE_BF16)
    return gkind == FMX_DTYPE_F32 ? launch_bits<__bf16, float, __bf16>(bits, grid, tab, sc, s)
                                  : launch_bits<__bf16, __bf16, __bf16>(bits, grid, tab, sc, s);
  if (ckind == FMX_DTYPE_F16) {
    if (gkind == FMX_DTYPE_F16) return launch_bits<float, _Float16, _Float16>(bits, grid, tab, sc, s);
    return launch_bits<float, float, _Float16>(bits, grid, tab, sc, s);
  }
  if (gkind == FMX_DTYPE_BF16) return launch_bits<float, __bf16, __bf16>(bits, grid, tab, sc, s);
  return launch_bits<float, float, __bf16>(bits, grid, tab, sc, s);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace

hipError_t launch_adamw(int pkind, int gkind, int ckind, int bits, const AdamWTensor* t, int64_t count,
                        const AdamWScalars& sc, hipStream_t s) {
  Table tab;
  tab.count = 0;
  int64_t grid = 0;
  auto flush = [&]() -> hipError_t {
    if (tab.count == 0) return hipSuccess;
    const hipError_t e = launch_types(pkind, gkind, ckind, bits, (int)grid, tab, sc, s);
    tab.count = 0;
    grid = 0;
    return e;
  };
  for (int64_t k = 0; k < count; ++k) {
    // a tensor of more workgroups than a launch's tail may hold goes on in pieces
    constexpr int64_t kPiece = (int64_t)1 << 20;  // workgroups
    for (int64_t at = 0; at < t[k].n; at += kPiece * kChunk) {
      const int64_t n = t[k].n - at < kPiece * kChunk ? t[k].n - at : kPiece * kChunk;
      if (tab.count == kMaxTensors || grid > kPiece) {
        const hipError_t e = flush();
        if (e != hipSuccess) return e;
      }
      const int ps = pkind == FMX_DTYPE_F32 ? 4 : 2, gs = gkind == FMX_DTYPE_F32 ? 4 : 2, ms = bits == 8 ? 1 : 4;
      const void* p[7] = {static_cast<char*>(t[k].param) + at * ps, static_cast<const char*>(t[k].grad) + at * gs,
                          static_cast<char*>(t[k].m) + at * ms,     static_cast<char*>(t[k].v) + at * ms,
                          t[k].ms ? t[k].ms + at / 256 : nullptr,   t[k].vs ? t[k].vs + at / 256 : nullptr,
                          t[k].copy ? static_cast<char*>(t[k].copy) + at * 2 : nullptr};
      const int mb = bits == 8 ? 8 : 16;
      const bool vec = aligned(p[0], 16) && aligned(p[1], 16) && aligned(p[2], mb) && aligned(p[3], mb) && aligned(p[6], 16);
      Entry& x = tab.t[tab.count];
      x.hi[0] = x.hi[1] = x.hi[2] = 0;
      x.hi[3] = vec ? 1u << 16 : 0u;
      for (int i = 0; i < 7; ++i) {
        const uint64_t v = reinterpret_cast<uint64_t>(p[i]);
        if (v >> 48) return hipErrorInvalidValue;
        x.lo[i] = (uint32_t)v;
        x.hi[i / 2] |= (uint32_t)(v >> 32) << (16 * (i & 1));
      }
      x.n = (uint32_t)n;
      tab.first[tab.count] = (int32_t)grid;
      grid += (n + kChunk - 1) / kChunk;
      tab.first[++tab.count] = (int32_t)grid;
    }
  }
  return flush();
}

hipError_t launch_adamw_decode(const void* codes, bool second, const float* scales, int64_t n, float* out,
                               hipStream_t s) {
  const int vec = aligned(codes, 8) && aligned(out, 16);
  constexpr int64_t kPiece = ((int64_t)1 << 30) * kElems;  // elements of a launch, a multiple of the block
  for (int64_t at = 0; at < n; at += kPiece) {
    const int64_t k = n - at < kPiece ? n - at : kPiece;
    const int grid = (int)((k + kThreads * kElems - 1) / (kThreads * kElems));
    const void* c = static_cast<const char*>(codes) + at;
    if (second)
      adamw_decode_kernel<true><<<grid, kThreads, 0, s>>>(c, scales + at / 256, k, out + at, vec);
    else
      adamw_decode_kernel<false><<<grid, kThreads, 0, s>>>(c, scales + at / 256, k, out + at, vec);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace fmx
