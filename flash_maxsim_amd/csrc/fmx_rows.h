// Pieces of 16 bytes of a row that may begin at any element and end early: the accesses need no more than an
// element's alignment here.
#pragma once

#include <hip/hip_runtime.h>

namespace fmx {
namespace {

// V consecutive elements of type T as they lie in memory.
template <typename T, int V>
struct Piece {
  T v[V];
  // `left` of them are there, the others are zeros
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, int left) {
    if (WHOLE ? left > 0 : left >= V) {
      __builtin_memcpy(v, p, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = T(0.0f);
      if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
          if (i < left) v[i] = p[i];
      }
    }
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(T* p, int left) const {
    if (WHOLE ? left > 0 : left >= V) {
      __builtin_memcpy(p, v, sizeof(v));
    } else if constexpr (!WHOLE) {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < left) p[i] = v[i];
    }
  }
};

}  // namespace
}  // namespace fmx
