// Pieces of 16 bytes of a row that may begin at any element and end early: the accesses need no more than an
// element's alignment here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fmx {
namespace {

// V consecutive elements of type T as they lie in memory. (They move as one vector: stores of the array itself, of
// zeros for one, came apart into stores of elements; 268 MB of zeros 160 us.)
template <typename T, int V>
struct Piece {
  typedef uint32_t words_t __attribute__((ext_vector_type(sizeof(T) * V / 4)));
  T v[V];
  // `left` of them are there, the others are zeros
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, int left) {
    words_t w = {};
    if (WHOLE ? left > 0 : left >= V) {
      __builtin_memcpy(&w, p, sizeof(w));
      set(w);
    } else {
      set(w);
      if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
          if (i < left) v[i] = p[i];
      }
    }
  }
  // PAST: past the caches, for what is too large to be found in them
  template <bool WHOLE, bool PAST = false>
  __device__ __forceinline__ void store(T* p, int left) const {
    if (WHOLE ? left > 0 : left >= V) {
      words_t w;
      __builtin_memcpy(&w, v, sizeof(w));
      if constexpr (PAST) {
        typedef words_t loose_t __attribute__((aligned(sizeof(T))));
        __builtin_nontemporal_store(w, reinterpret_cast<loose_t*>(p));
      } else {
        __builtin_memcpy(p, &w, sizeof(w));
      }
    } else if constexpr (!WHOLE) {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < left) p[i] = v[i];
    }
  }
  __device__ __forceinline__ void set(const words_t& w) { __builtin_memcpy(v, &w, sizeof(v)); }
};

}  // namespace
}  // namespace fmx
