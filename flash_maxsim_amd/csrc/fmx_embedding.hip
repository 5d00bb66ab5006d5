// Embedding lookup y[t] = scale W[ids[t]], and its gradient dW[v] = scale sum of dy[t] over the t with ids[t] = v.
//
// Bound by HBM: the lookup reads and writes T rows, the gradient reads T rows of dy and writes all V rows of dW.
//
// The gradient has no atomics on values: tokens are sorted by id (stable), so that the rows of an id lie in a fixed
// order, and the sorted list is cut into stretches of kStretch tokens whatever their ids: a wave sums a stretch's
// rows in registers and writes the ids that begin and end in it to dW; of an id that goes on past the
// stretch's end it writes a float32 partial sum, and a second kernel adds an id's partial sums in order. The sums so cost the
// same whatever ids repeat; the join does not, for an id's partial sums are a workgroup's for each 256 columns (100000 x 1024
// bf16, us of which the join, no id frequent / one id half of the tokens / all: 65536 tokens 104, 6 / 132, 31 / 145, 56;
// 2^20 tokens 665, 99 / 1108, 515 / 1719, 1095).
//
// Rows of ids that do not occur get zeros from workgroups of their own, beside the radix sort's few (which leave the GPU
// idle) or, where there is none, beside the sums. Which ids occur the first kernel notes: seen[id] is one of the
// id's tokens, whichever was stored last. The list is never cleared: an entry counts only if it names a token that has the id.
//
// Sorting: up to kRankMost tokens each counts the tokens before it (T^2 comparisons, one launch); more go through passes
// of a radix sort, of 2 launches each (3 of more than 2^18 tokens), by digits of up to 10 bits. Both for the whole gradient of a 30522 x 128 bf16 table,
// us: 1024 tokens 19 / 31, 4096 22 / 41, 8192 27 / 43, 12288 37 / 44, 16384 48 / 45.
//
// 65536 tokens of a 131072 x 1024 bf16 table, few ids most of the tokens, us: the lookup 41 (134 MB written, 3.3 TB/s, the
// few ids' rows out of the caches), the gradient 111: the sums 44 (134 MB of dy read row by row in the ids' order, 47 MB written,
// 4.1 TB/s), the sort 57, with 224 MB of zeros beside it, the join 9. 32 tokens of 768: the lookup 3.2, a launch's own time.
#include "fmx_device.h"
#include "fmx_layers.h"
#include "fmx_rows.h"

#include "../../include/fmx.h"

namespace fmx {
namespace {

constexpr int kStretch = 32;         // sorted tokens that a wave sums
constexpr int64_t kRankMost = 14336;
constexpr int kRows = 64;            // ids of a workgroup that writes zeros
constexpr int kBits = 10;            // of a digit, at most
constexpr int kTile = 4096;          // tokens of a workgroup of the radix sort
// A pass of more workgroups than this adds up their digits' counts in a launch of its own, fewer each for themselves, work that
// grows with their square (rows of 8 bf16 elements, 100000 ids, each for itself / a launch, us: 2^15 tokens 46 / 52, 2^17 55 / 60,
// 2^18 69 / 70, 2^19 98 / 95, 2^22 687 / 489, 2^24 5070 / 1810; 1000 ids, 2^26 tokens 81 ms / 6.2).
constexpr int kScanFrom = 64;
// A gradient of at least this many bytes is stored past the caches, which cannot hold it for its next reader (rows of 1024
// bf16 elements, the gradient alone and with a reader after it, us, through the caches / past them: 49152 rows 51 and 80 / 51
// and 82, 98304 59 and 135 / 65 and 141, 131072 118 and 209 / 92 and 195).
constexpr int64_t kPast = 224 << 20;

// The id of token t as a key of the sort: V for tokens without a gradient (outside 0 .. V - 1, or the padding id).
__device__ __forceinline__ int32_t key_of(const EmbeddingArgs& a, int64_t t) {
  const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[t] : (int64_t)static_cast<const int32_t*>(a.ids)[t];
  return id >= 0 && id < a.V && id != a.padding ? (int32_t)id : (int32_t)a.V;
}

// Where a lane's piece of V columns from `col` on begins. The last piece of an odd row begins at d - V and has some of the columns
// of the one before it: both lanes write the same there. (Rows that ended early, element by element, 65536 of 30522 x 771 fp16:
// lookup 41 us, gradient 82; now 34 and 64, and 31 and 61 of 768 columns.) Rows of less than a piece end early.
template <int V, bool WHOLE>
__device__ __forceinline__ int begin_of(int col, int d) {
  return !WHOLE && d >= V && col < d && col > d - V ? d - V : col;
}

// ---- lookup ----

// kAhead rows of a thread at a time: their ids, then their rows, then the stores, each in flight together. A workgroup's are
// neighbours (4096 x 1024 bf16 6.5 -> 4.4 us, 16384 x 768 11.0 -> 9.3, larger ones equal, against rows a launch apart).
constexpr int kAhead = 4;
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(256) embedding_kernel(EmbeddingArgs a, int lanes) {
  constexpr int V = 16 / sizeof(T), U = kAhead;
  const int lane = threadIdx.x & (lanes - 1), rows = 256 / lanes;
  for (int64_t t = (int64_t)blockIdx.x * rows * U + threadIdx.x / lanes; t < a.T; t += (int64_t)gridDim.x * rows * U) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = t + u * rows < a.T ? t + u * rows : t;
      id[u] = a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : (int64_t)static_cast<const int32_t*>(a.ids)[at];
    }
    for (int at = lane * V; at < a.d; at += lanes * V) {
      const int col = begin_of<V, WHOLE>(at, a.d);
      Piece<T, V> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        p[u].template load<WHOLE>(static_cast<const T*>(a.w) + (id[u] >= 0 && id[u] < a.V ? id[u] : 0) * a.sw + col, a.d - col);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = id[u] >= 0 && id[u] < a.V;
#pragma unroll
        for (int i = 0; i < V; ++i) p[u].v[i] = (T)(there ? (float)p[u].v[i] * a.scale : __builtin_nanf(""));
        if (t + u * rows < a.T) p[u].template store<WHOLE>(static_cast<T*>(a.out) + (t + u * rows) * a.d + col, a.d - col);
      }
    }
  }
}

// ---- rows of ids that do not occur ----

__device__ __forceinline__ void note(const EmbeddingArgs& a, int32_t key, int64_t t) {
  if (key < a.V) a.seen[key] = (int32_t)t;
}

// Zeros to the rows of kRows ids from v0 on that do not occur, by all threads of a workgroup.
template <int THREADS>
__device__ __forceinline__ void write_zeros(const EmbeddingArgs& a, int64_t v0) {
  __shared__ uint8_t absent[kRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x < kRows) {
    const int64_t v = v0 + threadIdx.x;
    // without tokens there is neither a list nor an id
    const int64_t t = v < a.V && a.T > 0 ? (int64_t)(uint32_t)a.seen[v] : a.T;
    absent[threadIdx.x] = v < a.V && (t >= a.T || key_of(a, t) != v);
  }
  __syncthreads();
  const int64_t bytes = (int64_t)a.d * a.size;
  for (int r = wave; r < kRows; r += THREADS / 64) {
    if (!absent[r]) continue;
    char* row = static_cast<char*>(a.out) + (v0 + r) * bytes;
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    if (a.past) {
      typedef u32x4_t loose_t __attribute__((aligned(2)));
      for (int64_t at = lane * 16; at + 16 <= bytes; at += 64 * 16)
        __builtin_nontemporal_store(zero, reinterpret_cast<loose_t*>(row + at));
    } else {
      for (int64_t at = lane * 16; at + 16 <= bytes; at += 64 * 16) __builtin_memcpy(row + at, &zero, 16);
    }
    const int64_t rest = bytes & ~(int64_t)15;  // elements of 2 or 4 bytes, a pair of bytes a lane
    if (rest + lane * 2 < bytes) *reinterpret_cast<uint16_t*>(row + rest + lane * 2) = 0;
  }
}

// ---- sorting ----

// Each token's place: how many come before it. A workgroup ranks 16 tokens; keys go through LDS, 4096 at a time. A wave
// compares its tokens (lane & 15) with 16 keys at a time, 4 for each group of 16 lanes; those before the workgroup's
// own 16 count where they are equal, too.
constexpr int kRankTile = 4096;
__global__ void __launch_bounds__(1024) embedding_rank_kernel(EmbeddingArgs a) {
  typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) int32_t keys[kRankTile];
  __shared__ int counts[16][64];
  const int lane = threadIdx.x & 63, group = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int T = (int)a.T, t0 = blockIdx.x * 16, t = t0 + (lane & 15);
  const int32_t mine = key_of(a, t < T ? t : T - 1);
  if (threadIdx.x < 16 && t < T) note(a, mine, t);
  int before = 0;
  for (int base = 0; base < T; base += kRankTile) {
    __syncthreads();
#pragma unroll
    for (int k = threadIdx.x; k < kRankTile; k += 1024) keys[k] = base + k < T ? key_of(a, base + k) : INT32_MAX;
    __syncthreads();
    const int end = T - base < kRankTile ? T - base : kRankTile;
    for (int k = wave * 16; k < end; k += 256) {
      const i32x4_t other = *reinterpret_cast<const i32x4_t*>(keys + k + 4 * group);
      const int at = base + k;  // uniform
      if (at == t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) before += other[i] < mine || (other[i] == mine && at + 4 * group + i < t) ? 1 : 0;
      } else {
        const int32_t bound = at < t0 ? mine + 1 : mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) before += other[i] < bound ? 1 : 0;
      }
    }
  }
  counts[wave][lane] = before;
  __syncthreads();
  if (threadIdx.x < 16 && t < T) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
#pragma unroll
      for (int g = 0; g < 4; ++g) place += counts[w][g * 16 + threadIdx.x];
    a.keys[place] = mine;
    a.order[place] = t;
  }
}

// One pass of the radix sort: the key's bits `shift` .. shift + bits - 1. FIRST: keys come from the ids.
template <bool FIRST>
__global__ void __launch_bounds__(1024) embedding_count_kernel(EmbeddingArgs a, int shift, int bits, const int32_t* keys,
                                                              int32_t* counts) {
  __shared__ int32_t hist[1 << kBits];
  const int digits = 1 << bits;
  if ((int)threadIdx.x < digits) hist[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTile / 1024; ++k) {
    const int64_t t = (int64_t)blockIdx.x * kTile + k * 1024 + threadIdx.x;
    if (t >= a.T) break;
    const int32_t key = FIRST ? key_of(a, t) : keys[t];
    if (FIRST) note(a, key, t);
    atomicAdd(&hist[(key >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x < digits) counts[(int64_t)blockIdx.x * digits + threadIdx.x] = hist[threadIdx.x];
}

// The counts of each digit, [groups][digits], to those of the workgroups before, and their sum to the row behind them. A
// workgroup has 32 digits, its threads 32 stretches of the groups.
__global__ void __launch_bounds__(1024) embedding_scan_kernel(int32_t* counts, int groups, int digits) {
  __shared__ int32_t sums[32][33];
  const int digit = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  const int per = (groups + 31) / 32, from = part * per, end = from + per < groups ? from + per : groups;
  int sum = 0;
  if (digit < digits) {
#pragma unroll 8
    for (int g = from; g < end; ++g) sum += counts[(int64_t)g * digits + digit];
  }
  sums[part][threadIdx.x & 31] = sum;
  __syncthreads();
  if (digit >= digits) return;
  int before = 0;
  for (int p = 0; p < part; ++p) before += sums[p][threadIdx.x & 31];
  constexpr int U = 8;  // counts in flight
  for (int g = from; g < end; g += U) {
    int n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) n[u] = g + u < end ? counts[(int64_t)(g + u) * digits + digit] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g + u < end) counts[(int64_t)(g + u) * digits + digit] = before;
      before += n[u];
    }
  }
  if (part == 31) counts[(int64_t)groups * digits + digit] = before;
}

// Tokens to their places of this pass, in their order before it: digits before, workgroups before, waves before (a
// wave has kTile / 16 neighbouring tokens), tokens of the wave before. The workgroups after those of the tokens write
// zeros, to the ids from `zeros` on.
template <bool FIRST>
__global__ void __launch_bounds__(1024) embedding_place_kernel(EmbeddingArgs a, int shift, int bits, const int32_t* keys,
                                                              const int32_t* order, const int32_t* counts, int groups,
                                                              int32_t* keys_out, int32_t* order_out, int64_t zeros) {
  if ((int)blockIdx.x >= groups) return write_zeros<1024>(a, zeros + (int64_t)((int)blockIdx.x - groups) * kRows);
  __shared__ int32_t mine[16][1 << kBits];
  __shared__ int32_t sums[16];
  const int digits = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // how many tokens lie before this workgroup's of digit threadIdx.x
  int total = 0, before = 0;
  if ((int)threadIdx.x < digits && groups > kScanFrom) {
    total = counts[(int64_t)groups * digits + threadIdx.x];
    before = counts[(int64_t)blockIdx.x * digits + threadIdx.x];
  } else if ((int)threadIdx.x < digits) {
#pragma unroll 8
    for (int g = 0; g < groups; ++g) {
      const int n = counts[(int64_t)g * digits + threadIdx.x];
      total += n;
      before += g < (int)blockIdx.x ? n : 0;
    }
  }
  int scan = total;  // up to and with this digit
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const int other = __shfl_up(scan, k);
    scan += lane >= k ? other : 0;
  }
  if (lane == 63) sums[wave] = scan;
  for (int k = threadIdx.x; k < 16 * digits; k += 1024) mine[k / digits][k & (digits - 1)] = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) before += sums[w];
  before += scan - total;

  constexpr int kRounds = kTile / 1024;
  int32_t key[kRounds], from[kRounds];
  int place[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t t = (int64_t)blockIdx.x * kTile + wave * (kTile / 16) + k * 64 + lane;
    const bool there = t < a.T;
    key[k] = there ? (FIRST ? key_of(a, t) : keys[t]) : 0;
    from[k] = there ? (FIRST ? (int32_t)t : order[t]) : 0;
    const int digit = (key[k] >> shift) & (digits - 1);
    uint64_t same = __ballot(there);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((digit >> b) & 1);
      same &= (digit >> b) & 1 ? set : ~set;
    }
    const int ahead = __popcll(same & (((uint64_t)1 << lane) - 1));
    place[k] = there ? mine[wave][digit] + ahead : -1;
    // the wave's lanes have read the count; the last of each digit moves it on
    __builtin_amdgcn_wave_barrier();
    if (there && (same >> lane) == 1) mine[wave][digit] = place[k] + 1;
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if ((int)threadIdx.x < digits) {
    int at = before;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int n = mine[w][threadIdx.x];
      mine[w][threadIdx.x] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    if (place[k] < 0) continue;
    const int to = mine[wave][(key[k] >> shift) & (digits - 1)] + place[k];
    keys_out[to] = key[k];
    order_out[to] = from[k];
  }
}

// ---- sums ----

// Workgroups before `sums` add up stretches, a wave a stretch of one block of 64 pieces of columns; the others write
// the rows of ids that do not occur, kRows ids each.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(256) embedding_sum_kernel(EmbeddingArgs a, uint32_t sums, int blocks) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  T* out = static_cast<T*>(a.out);
  if (blockIdx.x >= sums) return write_zeros<256>(a, (int64_t)(blockIdx.x - sums) * kRows);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave, stretch = id / blocks;
  const int col = begin_of<V, WHOLE>((int)(id - stretch * blocks) * 64 * V + lane * V, a.d);
  const int64_t from = stretch * kStretch;
  if (from >= a.T) return;
  const int n = a.T - from < kStretch ? (int)(a.T - from) : kStretch;
  const int32_t k = lane < n ? a.keys[from + lane] : (int32_t)a.V, t = lane < n ? a.order[from + lane] : 0;
  const int32_t last = from > 0 ? a.keys[from - 1] : -1, next = from + n < a.T ? a.keys[from + n] : -1;
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0f;
  const T* dy = static_cast<const T*>(a.dy);
  constexpr int U = 8;  // rows in flight
  Piece<T, V> p[U];
  auto load = [&](int at) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = __builtin_amdgcn_readlane(t, at + u < n ? at + u : n - 1);
      p[u].template load<WHOLE>(dy + row * a.sdy + col, a.d - col);
    }
  };
  for (int at = 0; at < n; at += U) {
    load(at);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at + u >= n) break;
      const int32_t key = __builtin_amdgcn_readlane(k, at + u);
      if (key >= a.V) return;  // tokens without a gradient come last
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += (float)p[u].v[i];
      const int32_t after = at + u + 1 < n ? __builtin_amdgcn_readlane(k, at + u + 1) : next;
      if (after == key && at + u + 1 < n) continue;
      const bool begins = __builtin_amdgcn_readlane(k, 0) != key || last != key, ends = after != key;
      if (col < a.d) {
        if (begins && ends) {
          Piece<T, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) o.v[i] = (T)(s[i] * a.scale);
          if (a.past)
            o.template store<WHOLE, true>(out + (int64_t)key * a.d + col, a.d - col);
          else
            o.template store<WHOLE>(out + (int64_t)key * a.d + col, a.d - col);
        } else {
          // an id that goes on: its first stretch's sum in slot 1, the later ones' in slot 0
          typedef f32x4_t loose_t __attribute__((aligned(4)));
          float* part = a.part + ((stretch * 2 + (begins ? 1 : 0)) * blocks) * 64 * V + col;
#pragma unroll
          for (int i = 0; i < V; i += 4)
            *reinterpret_cast<loose_t*>(part + i) = f32x4_t{s[i], s[i + 1], s[i + 2], s[i + 3]};
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = 0.0f;
    }
  }
}

// Ids that go past a stretch's end: a wave for each stretch that such an id may begin in, and 256 columns, adds the id's
// partial sums. Those of more than kLong the sixteen waves of a workgroup add together, every sixteenth each, and then
// the waves' sums.
constexpr int kLong = 24;
template <typename T>
__global__ void __launch_bounds__(1024) embedding_join_kernel(EmbeddingArgs a, int pitch) {
  __shared__ __attribute__((aligned(16))) f32x4_t sums[16][64];
  __shared__ int64_t longs[16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t stretch = (int64_t)blockIdx.x * 16 + wave, end = (stretch + 1) * kStretch;
  const int col = blockIdx.y * 256 + lane * 4;
  // the stretches after this one that begin with the id that goes on from it; 0: none begins here and goes on
  int64_t more = 0;
  int32_t key = 0;
  if (end < a.T) {
    const int32_t first = a.keys[stretch * kStretch], last = stretch > 0 ? a.keys[stretch * kStretch - 1] : -1,
                  next = a.keys[end];
    key = a.keys[end - 1];
    if (key < a.V && next == key && !(first == key && last == key)) {
      for (;;) {
        const int64_t at = (stretch + 1 + more + lane) * kStretch;
        const uint64_t same = __ballot(at < a.T && a.keys[at < a.T ? at : 0] == key);
        const int n = same == ~(uint64_t)0 ? 64 : __builtin_ctzll(~same);
        more += n;
        if (n < 64) break;
      }
    }
  }
  // every `step`-th partial sum of an id that begins in stretch `at`, from number q on
  auto add = [&](int64_t at, int64_t q, int64_t more, int step) {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
    if (col < pitch) {
      const float* part = a.part + col;
#pragma unroll 4
      for (; q <= more; q += step)
        s += *reinterpret_cast<const f32x4_t*>(part + ((at + q) * 2 + (q == 0 ? 1 : 0)) * pitch);
    }
    return s;
  };
  auto write = [&](int32_t key, const f32x4_t& s) {
    T* out = static_cast<T*>(a.out) + (int64_t)key * a.d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < a.d) out[col + i] = (T)(s[i] * a.scale);
  };
  if (more > 0 && more <= kLong) write(key, add(stretch, 0, more, 1));
  if (lane == 0) longs[wave] = more > kLong ? more : 0;
  __syncthreads();
  for (int k = 0; k < 16; ++k) {
    const int64_t n = longs[k];
    if (n == 0) continue;
    const int64_t at = (int64_t)blockIdx.x * 16 + k;
    f32x4_t s = add(at, wave, n, 16);
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < 16; ++w) s += sums[w][lane];
      write(a.keys[at * kStretch + kStretch - 1], s);
    }
    __syncthreads();
  }
}

template <typename T>
hipError_t lookup(const EmbeddingArgs& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  int lanes = 1;
  while (lanes < 256 && lanes * V < a.d) lanes *= 2;
  const int64_t rows = 256 / lanes, want = (a.T + rows * kAhead - 1) / (rows * kAhead), most = (int64_t)layer_cus() * 16;
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (a.d % V == 0)
    embedding_kernel<T, true><<<grid, 256, 0, s>>>(a, lanes);
  else
    embedding_kernel<T, false><<<grid, 256, 0, s>>>(a, lanes);
  return hipGetLastError();
}

int bits_of(int64_t V) {  // of the keys 0 .. V
  int bits = 1;
  while (V >> bits) ++bits;
  return bits;
}

int64_t stretches_of(int64_t T) { return (T + kStretch - 1) / kStretch; }

struct Layout {
  int64_t keys, counts, seen, part, total;  // bytes: lists of keys and of tokens; digits' counts; partial sums
};
Layout layout(int kind, int64_t T, int64_t V, int64_t d) {
  const int64_t per = 64 * (kind == FMX_DTYPE_F32 ? 4 : 8), pitch = (d + per - 1) / per * per;
  const bool radix = T > kRankMost;
  Layout l;
  l.keys = (T * 4 + 255) / 256 * 256;
  l.counts = radix ? ((T + kTile - 1) / kTile + 1) * (4 << kBits) : 0;
  l.seen = T ? (V * 4 + 255) / 256 * 256 : 0;
  l.part = stretches_of(T) * 2 * pitch * 4;
  l.total = (radix ? 4 : 2) * l.keys + l.counts + l.seen + l.part;
  return l;
}

template <typename T>
hipError_t gradient(int kind, EmbeddingArgs a, char* ws, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const Layout l = layout(kind, a.T, a.V, a.d);
  int32_t* lists[4];
  for (int i = 0; i < 4; ++i) lists[i] = reinterpret_cast<int32_t*>(ws + (i < 2 || a.T > kRankMost ? i * l.keys : 0));
  a.keys = lists[0];
  a.order = lists[1];
  a.seen = reinterpret_cast<int32_t*>(ws + l.total - l.part - l.seen);
  a.size = (int)sizeof(T);
  a.past = a.V * a.d * a.size >= kPast;
  const int64_t rows = (a.V + kRows - 1) / kRows;  // workgroups that write zeros
  if (a.T > kRankMost) {
    int32_t* counts = reinterpret_cast<int32_t*>(ws + 4 * l.keys);
    const int bits = bits_of(a.V), passes = (bits + kBits - 1) / kBits, groups = (int)((a.T + kTile - 1) / kTile);
    int shift = 0;
    for (int p = 0; p < passes; ++p) {  // the bits left over the passes left
      const int b = (bits - shift + passes - p - 1) / (passes - p), to = (p & 1) * 2, from = 2 - to;
      const int64_t z0 = rows * p / passes, zn = rows * (p + 1) / passes - z0;
      const unsigned grid = (unsigned)(groups + zn);
      if (p == 0)
        embedding_count_kernel<true><<<groups, 1024, 0, s>>>(a, shift, b, nullptr, counts);
      else
        embedding_count_kernel<false><<<groups, 1024, 0, s>>>(a, shift, b, lists[from], counts);
      if (groups > kScanFrom)
        embedding_scan_kernel<<<(unsigned)(((1 << b) + 31) / 32), 1024, 0, s>>>(counts, groups, 1 << b);
      if (p == 0)
        embedding_place_kernel<true>
            <<<grid, 1024, 0, s>>>(a, shift, b, nullptr, nullptr, counts, groups, lists[to], lists[to + 1], z0 * kRows);
      else
        embedding_place_kernel<false>
            <<<grid, 1024, 0, s>>>(a, shift, b, lists[from], lists[from + 1], counts, groups, lists[to], lists[to + 1],
                                   z0 * kRows);
      a.keys = lists[to];
      a.order = lists[to + 1];
      shift += b;
    }
  } else if (a.T > 0) {
    embedding_rank_kernel<<<(unsigned)((a.T + 15) / 16), 1024, 0, s>>>(a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  a.part = reinterpret_cast<float*>(ws + l.total - l.part);
  const int blocks = (int)((a.d + 64 * V - 1) / (64 * V));
  const uint32_t sums = (uint32_t)((stretches_of(a.T) * blocks + 3) / 4);
  const uint32_t grid = sums + (a.T > kRankMost ? 0u : (uint32_t)rows);
  if (a.d % V == 0)
    embedding_sum_kernel<T, true><<<grid, 256, 0, s>>>(a, sums, blocks);
  else
    embedding_sum_kernel<T, false><<<grid, 256, 0, s>>>(a, sums, blocks);
  e = hipGetLastError();
  if (e != hipSuccess || a.T <= kStretch) return e;
  embedding_join_kernel<T><<<dim3((unsigned)((stretches_of(a.T) + 14) / 16), (unsigned)((a.d + 255) / 256)), 1024, 0, s>>>(
      a, blocks * 64 * V);
  return hipGetLastError();
}

}  // namespace

size_t embedding_workspace_bytes(int kind, int64_t T, int64_t V, int64_t d) { return (size_t)layout(kind, T, V, d).total; }

hipError_t launch_embedding(int kind, const EmbeddingArgs& a, hipStream_t s) {
  if (kind == FMX_DTYPE_F32) return lookup<float>(a, s);
  if (kind == FMX_DTYPE_BF16) return lookup<__bf16>(a, s);
  return lookup<_Float16>(a, s);
}

hipError_t launch_embedding_bwd(int kind, const EmbeddingArgs& a, void* ws, hipStream_t s) {
  if (kind == FMX_DTYPE_F32) return gradient<float>(kind, a, static_cast<char*>(ws), s);
  if (kind == FMX_DTYPE_BF16) return gradient<__bf16>(kind, a, static_cast<char*>(ws), s);
  return gradient<_Float16>(kind, a, static_cast<char*>(ws), s);
}

}  // namespace fmx
