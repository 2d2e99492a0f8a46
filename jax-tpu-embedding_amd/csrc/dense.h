// Device helpers of the dense operators (layer_norm.hip, experts.hip,
// adamw.hip): element types, vectors of them, and sums over lanes.
#pragma once

#include "../../include/scemb.h"
#include "common.h"

namespace scemb {

using bf16 = __bf16;
using f16 = _Float16;

// V consecutive elements, loaded and stored with one instruction of up to 16
// bytes. It is aligned as its elements are, no more: gfx950 takes wide loads
// and stores at any address, so rows of any length and start are moved 16 bytes
// a lane (the sum of four rows of 1975 float32 for each of 7084 tokens: 61 us,
// element by element 127).
template <typename T, int V>
struct Vec {
  T v[V];
};

// A vector's bytes as one value, aligned to 2 bytes as the smallest elements
// are.
template <int kBytes>
struct Words;
template <>
struct Words<16> {
  typedef uint32_t Vector __attribute__((ext_vector_type(4)));
  typedef Vector Type __attribute__((aligned(2)));
};
template <>
struct Words<8> {
  typedef uint32_t Vector __attribute__((ext_vector_type(2)));
  typedef Vector Type __attribute__((aligned(2)));
};

// Elements of 16 bytes.
template <typename T>
constexpr int kVec = 16 / sizeof(T);

// kStream: memory that is not touched again soon; the access leaves other data
// in the caches.
template <typename T, int V, bool kStream = false>
__device__ __forceinline__ Vec<T, V> LoadVec(const T* p) {
  if constexpr (kStream) {
    using W = Words<sizeof(T) * V>;
    return __builtin_bit_cast(
        Vec<T, V>, __builtin_nontemporal_load(
                       reinterpret_cast<const typename W::Type*>(p)));
  } else {
    return *reinterpret_cast<const Vec<T, V>*>(p);
  }
}
template <typename T, int V, bool kStream = false>
__device__ __forceinline__ void StoreVec(T* p, const Vec<T, V>& x) {
  if constexpr (kStream) {
    using W = Words<sizeof(T) * V>;
    __builtin_nontemporal_store(__builtin_bit_cast(typename W::Type, x),
                                reinterpret_cast<typename W::Type*>(p));
  } else {
    *reinterpret_cast<Vec<T, V>*>(p) = x;
  }
}

// How rows of a length are cut into vectors of V elements.
enum class Cut {
  kWhole,  // the length is a multiple of V
  kOver,   // above V: the last vector ends at the row's end and repeats
           // elements of the one before it
  kPart,   // below V: one vector, of which `dim` elements exist
};

// The vector of a row at element c < dim: where it starts, and its elements
// [lo, hi) that no other vector has. Repeated elements hold and get the same
// values twice; only sums leave them out. (An element-wise end of the row
// instead costs every wavefront a second wait for memory.)
template <Cut kCut, int V>
struct Span {
  int at;
  int lo;
  int hi;

  __device__ __forceinline__ Span(int c, int dim)
      : at(kCut == Cut::kOver && c > dim - V ? dim - V : c),
        lo(c - at),
        hi(kCut == Cut::kPart ? dim : V) {}

  // Whether element j counts.
  __device__ __forceinline__ bool Has(int j) const {
    return kCut == Cut::kWhole || (kCut == Cut::kOver ? j >= lo : j < hi);
  }
};

// Elements [p, p + V), zero past the end of a row of less.
template <Cut kCut, typename T, int V, bool kStream = false>
__device__ __forceinline__ Vec<T, V> LoadSpan(const T* row,
                                              const Span<kCut, V>& s) {
  if constexpr (kCut != Cut::kPart) {
    return LoadVec<T, V, kStream>(row + s.at);
  }
  Vec<T, V> x;
#pragma unroll
  for (int j = 0; j < V; ++j) x.v[j] = j < s.hi ? row[j] : static_cast<T>(0);
  return x;
}
template <Cut kCut, typename T, int V>
__device__ __forceinline__ void StoreSpan(T* row, const Span<kCut, V>& s,
                                          const Vec<T, V>& x) {
  if constexpr (kCut != Cut::kPart) {
    StoreVec<T, V>(row + s.at, x);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j < s.hi) row[j] = x.v[j];
    }
  }
}

// Calls of layer norm's gradient (rows in registers), of the rows to their
// experts and back, and of AdamW that move more than the last cache holds (256
// MB) read past it what they read once (the other kernels were not timed that
// way): 65,536 x 1024 bfloat16 backwards through layer norm 80 us
// through the caches, 74 past them, the sum of two rows of 1024 for each of
// 65,536 tokens 77 and 66; but 16,384 x 1024 24 and 27, and 20,011 tokens 20 and
// 25. Results are always written through the caches, for whoever reads them
// next (past them, a product or an activation that follows takes 1 to 8% longer
// than the write saves).
constexpr int64_t kCacheBytes = 256 << 20;

inline Cut CutOf(int64_t dim, int v) {
  return dim % v == 0 ? Cut::kWhole : dim > v ? Cut::kOver : Cut::kPart;
}

// ---------------------------------------------------------------------------
// Sums over G neighbouring lanes (G a power of two up to 64); every lane gets
// the sum. Steps within 16 lanes are DPP moves, the last two the lane swaps
// of gfx950: no LDS traffic. Each step adds the same two partial sums in both
// lanes, so all lanes hold the same bits.
// ---------------------------------------------------------------------------

template <int kCtrl>
__device__ __forceinline__ float DppMove(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), kCtrl, 0xf,
                                      0xf, true));
}

constexpr int kDppXor1 = 0xb1;         // quad_perm [1, 0, 3, 2]
constexpr int kDppXor2 = 0x4e;         // quad_perm [2, 3, 0, 1]
constexpr int kDppHalfMirror = 0x141;  // lane i of 8 <- lane 7 - i
constexpr int kDppMirror = 0x140;      // lane i of 16 <- lane 15 - i

struct LaneAdd {
  static __device__ __forceinline__ float Of(float a, float b) {
    return a + b;
  }
};
// The larger of two values that are not negative, as bit patterns: a NaN is
// above every number and stays.
struct LaneMaxBits {
  static __device__ __forceinline__ float Of(float a, float b) {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a),
                                         __builtin_bit_cast(uint32_t, b)));
  }
};

template <typename Op, int G>
__device__ __forceinline__ float LaneReduce(float x) {
  static_assert(G >= 1 && G <= kWave && (G & (G - 1)) == 0, "power of two");
  if constexpr (G >= 2) x = Op::Of(x, DppMove<kDppXor1>(x));
  if constexpr (G >= 4) x = Op::Of(x, DppMove<kDppXor2>(x));
  if constexpr (G >= 8) x = Op::Of(x, DppMove<kDppHalfMirror>(x));
  if constexpr (G >= 16) x = Op::Of(x, DppMove<kDppMirror>(x));
  if constexpr (G >= 32) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    // Copies: a bit cast of a vector's element reads element 0.
    const uint32_t lo = r[0], hi = r[1];
    x = Op::Of(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
  }
  if constexpr (G >= 64) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    // Copies: a bit cast of a vector's element reads element 0.
    const uint32_t lo = r[0], hi = r[1];
    x = Op::Of(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
  }
  return x;
}

template <int G>
__device__ __forceinline__ float LaneSum(float x) {
  return LaneReduce<LaneAdd, G>(x);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Work-groups of a launch at most: a grid has fewer than 2^32 threads.
constexpr int64_t MostGroups(int threads) { return 0xffffffffll / threads; }

inline int TypeBytes(int32_t type) {
  return type == SCEMB_F32 ? 4
         : type == SCEMB_BF16 || type == SCEMB_F16 ? 2
                                                   : 0;
}

}  // namespace scemb
