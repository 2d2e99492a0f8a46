// Device helpers of the matrix products (expert_matmul.hip, matmul_8bit.hip):
// matrix instructions, panels of an operand in LDS, and the tile of a
// work-group.
#pragma once

#include "dense.h"

namespace scemb {

using F32x16 = float __attribute__((ext_vector_type(16)));
using U32x4 = uint32_t __attribute__((ext_vector_type(4)));

using LdsBytes = __attribute__((address_space(3))) void*;

// Memory from a pointer on that is the same for all lanes. Lanes add 32 bits,
// which stay in registers of their own: a register that held an address and is
// written again first waits for the load.
struct Memory {
  __amdgpu_buffer_rsrc_t rsrc;

  explicit __device__ __forceinline__ Memory(const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint64_t at =
        static_cast<uint64_t>(static_cast<uint32_t>(
            __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32))))
            << 32 |
        static_cast<uint32_t>(
            __builtin_amdgcn_readfirstlane(static_cast<int>(v)));
    rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(at), 0,
                                             0xffffffff, 0x00020000);
  }
  // 16 bytes a lane straight to LDS; the wavefront's land one after another
  // from `lds` on, which is the same for all its lanes.
  __device__ __forceinline__ void ToLds(uint32_t offset, char* lds) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsBytes)lds, 16,
                                             static_cast<int>(offset), 0, 0,
                                             0);
  }
};

// No memory access moves across, and all of this wavefront's loads have landed
// but the last `kNewer`.
template <int kNewer>
__device__ __forceinline__ void WaitLoads() {
  static_assert(kNewer >= 0 && kNewer < 64, "a count of six bits");
  asm volatile("" ::: "memory");
  // vmcnt in bits [3:0] and [15:14], the other counters at their largest.
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kNewer & 15) | (kNewer >> 4) << 14);
  asm volatile("" ::: "memory");
}

// All wavefronts of the work-group are here; LDS that they read before is free,
// what they waited for is in LDS.
__device__ __forceinline__ void Barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): LDS accesses are done
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------
// Panels: `kOuter` rows or columns of an operand by 128 bytes of the sum's index
// ("depth"), in LDS.
//
// kDepth: neighbours in memory are neighbours along the depth. A row is 128
// bytes, a line of the caches (of 64 bytes, every line came from L2 twice), its
// eight 16-byte chunks permuted so that 16 lanes that read one chunk of 16 rows
// find them in different banks (of 64).
// kOuter: neighbours in memory are neighbours along the outer index. LDS holds
// a row for each depth index, its chunks permuted by the depth index; reading
// transposes (16 bits) or gathers (32 bits).
// ---------------------------------------------------------------------------

enum class Along { kDepth, kOuter };

// x without its first `bytes` bytes (an even number up to 16), zeros behind.
__device__ __forceinline__ U32x4 ShiftDown(U32x4 x, int bytes) {
  if (bytes & 16) x = U32x4{0, 0, 0, 0};
  if (bytes & 8) x = U32x4{x[2], x[3], 0, 0};
  if (bytes & 4) x = U32x4{x[1], x[2], x[3], 0};
  if (bytes & 2) {
    x = U32x4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16,
              x[2] >> 16 | x[3] << 16, x[3] >> 16};
  }
  return x;
}

template <typename T, Along kAlong, int kOuter, int kThreads>
struct Panel {
  static constexpr int kBytes = kOuter * 128;
  static constexpr int kDepth = 128 / sizeof(T);
  static constexpr int kEach = 16 / sizeof(T);  // elements of a chunk
  // Threads that load a panel; where it has fewer chunks than threads, several
  // wavefronts load the same ones to the same places, and every wavefront has
  // the same number of loads to wait for.
  static constexpr int kLoaders =
      kBytes / 16 < kThreads ? kBytes / 16 : kThreads;
  static constexpr int kPer = kBytes / 16 / kLoaders;  // chunks of a thread
  static constexpr int kRowChunks =
      kAlong == Along::kDepth ? 8 : kOuter * sizeof(T) / 16;
  static_assert(kPer * 16 * kLoaders == kBytes && kLoaders % kWave == 0 &&
                    kThreads % kLoaders == 0,
                "whole chunks");
  static_assert(kLoaders % kRowChunks == 0, "a thread's chunks share a column");

  // What chunk numbers of LDS row `row` are XORed with.
  static __device__ __forceinline__ int Key(int row) {
    if constexpr (kAlong == Along::kDepth) return (row >> 1) & 7;
    if constexpr (sizeof(T) == 4) {
      // Lanes of two rows 4 apart read 128 bytes each.
      return ((row >> 2) & 1) * 8 & (kRowChunks - 1);
    }
    // Lanes of rows 0-3, and of those 8 later, read 64 bytes each.
    return (((row & 3) | ((row >> 3) & 1) << 2) << 2) & (kRowChunks - 1);
  }

  // The thread's chunk i: its row in LDS, and which chunk of that row in
  // memory.
  static __device__ __forceinline__ int Row(int i) {
    return i * (kLoaders / kRowChunks) + threadIdx.x % kLoaders / kRowChunks;
  }
  static __device__ __forceinline__ int Column(int i) {
    return (threadIdx.x % kRowChunks) ^ Key(Row(i));
  }
  static __device__ __forceinline__ char* Place(char* lds, int i) {
    const int wave =
        __builtin_amdgcn_readfirstlane(threadIdx.x % kLoaders / kWave);
    return lds + (i * kLoaders + wave * kWave) * 16;
  }

  // --- Straight to LDS: chunks are aligned, and none ends past the last
  // element. ---

  uint32_t offset[kPer];  // of chunk i from the panel's first element, bytes

  // outer >= 1: the outer indices that exist. Others get some that do, and
  // their results are not stored.
  __device__ __forceinline__ void Start(int64_t stride, int outer) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if constexpr (kAlong == Along::kDepth) {
        offset[i] = static_cast<uint32_t>(min(Row(i), outer - 1)) *
                        static_cast<uint32_t>(stride * sizeof(T)) +
                    Column(i) * 16;
      } else {
        const int c = Column(i);
        offset[i] = static_cast<uint32_t>(Row(i)) *
                        static_cast<uint32_t>(stride * sizeof(T)) +
                    (c * kEach < outer ? c : 0) * 16;
      }
    }
  }

  // All of the panel's depth exists.
  __device__ __forceinline__ void Load(const char* from, char* lds) const {
    const Memory memory(from);
#pragma unroll
    for (int i = 0; i < kPer; ++i) memory.ToLds(offset[i], Place(lds, i));
  }

  // --- Through registers: any alignment, any number of elements (kWhole: whole
  // chunks). ---

  struct Chunks {
    U32x4 v[kPer];
    int drop[kPer];  // bytes at the start that are not the chunk's
  };
  // `total`: elements of a whole row in memory (where kAlong is kDepth, of the
  // whole depth). Chunks that reach past a row's end are loaded up to there, and
  // shifted when they are put into LDS: no element by itself, no branch and no
  // wait, so that a thread's loads are all under way while a step is multiplied.
  template <bool kWhole>
  static __device__ __forceinline__ void Fetch(const T* from, int64_t stride,
                                               int outer, int left,
                                               int32_t total, Chunks* to) {
    const int along = kAlong == Along::kDepth ? left : outer;
    const int rows = kAlong == Along::kDepth ? outer : left;
    if (kWhole || total >= kEach) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = Column(i) * kEach, row = Row(i);
        const int have = row < rows ? min(max(along - c, 0), kEach) : 0;
        // With nothing there: the first row's first elements, or, in a panel
        // that begins close to the row's end, its last.
        const T* p = have > 0 ? from + row * stride + (c + have - kEach)
                              : from + min(0, along - kEach);
        to->v[i] = __builtin_bit_cast(U32x4, LoadVec<T, kEach>(p));
        to->drop[i] = (kEach - have) * static_cast<int>(sizeof(T));
      }
    } else if constexpr (!kWhole) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = Column(i) * kEach, row = Row(i);
        const int have = row < rows ? along - c : 0;
        Vec<T, kEach> x;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          x.v[j] = j < have ? from[row * stride + c + j] : static_cast<T>(0.f);
        }
        to->v[i] = __builtin_bit_cast(U32x4, x);
        to->drop[i] = 0;
      }
    }
  }
  static __device__ __forceinline__ void Put(const Chunks& from, char* lds) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      *reinterpret_cast<U32x4*>(
          lds + (i * kLoaders + threadIdx.x % kLoaders) * 16) =
          ShiftDown(from.v[i], from.drop[i]);
    }
  }

  // --- Fragments: 32 outer indices from `outer` on by a quarter of the depth.
  // A lane gets outer index lane % 32 and 16 bytes of depth, from element
  // (2 * quarter + lane / 32) * kEach on. The panel begins `first` bytes into
  // `lds`. (An address is the array and one sum: the compiler follows no long
  // chain to the array, and would wait for loads into other ones.) ---

  static __device__ __forceinline__ U32x4 Fragment(const char* lds, int first,
                                                   int outer, int quarter) {
    const int lane = threadIdx.x % kWave;
    const int i = lane % 32, chunk = quarter * 2 + lane / 32;
    if constexpr (kAlong == Along::kDepth) {
      const int at = first + (outer + i) * 128 + ((chunk ^ Key(i)) * 16);
      return *reinterpret_cast<const U32x4*>(lds + at);
    } else if constexpr (sizeof(T) == 4) {
      U32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = chunk * 4 + j;
        const int c = ((outer + i) / 4) ^ Key(row);
        const int at = first + row * (kRowChunks * 16) + c * 16 + (i % 4) * 4;
        v[j] = *reinterpret_cast<const uint32_t*>(lds + at);
      }
      return v;
    } else {
      // Four lanes address four neighbours each of one depth index, 16 lanes
      // four depth indices; lane j of the 16 gets the four of outer index j.
      using S16x4 = short __attribute__((ext_vector_type(4)));
      using S16x4Lds = __attribute__((address_space(3))) S16x4;
      const int in = lane % 16, from = outer + lane / 16 % 2 * 16;
      uint2 part[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = chunk * 8 + j * 4 + in / 4;
        const int c = (from / 8 + in % 4 / 2) ^ Key(row);
        const int at = first + row * (kRowChunks * 16) + c * 16 + in % 2 * 8;
        part[j] = __builtin_bit_cast(
            uint2,
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((S16x4Lds*)(lds + at)));
      }
      return U32x4{part[0].x, part[0].y, part[1].x, part[1].y};
    }
  }
};

// acc[n][m] += the sum over a quarter of b[n] * a[m], for 32 of each. A lane
// holds m = lane % 32 and n = 8 * (i / 4) + 4 * (lane / 32) + i % 4 in element i.
template <typename T>
__device__ __forceinline__ void MultiplyAdd(const U32x4& b, const U32x4& a,
                                            F32x16* acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t bj = b[j], aj = a[j];
      *acc = __builtin_amdgcn_mfma_f32_32x32x2f32(
          __builtin_bit_cast(float, bj), __builtin_bit_cast(float, aj), *acc,
          0, 0, 0);
    }
  } else if constexpr (__is_same(T, bf16)) {
    using V = bf16 __attribute__((ext_vector_type(8)));
    *acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(V, b), __builtin_bit_cast(V, a), *acc, 0, 0, 0);
  } else {
    using V = f16 __attribute__((ext_vector_type(8)));
    *acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(V, b), __builtin_bit_cast(V, a), *acc, 0, 0, 0);
  }
}

// 8-bit operands (e4m3), whose values of a block share a power of two. They are
// multiplied as bfloat16, whose products are exact and whose sums are float32's:
// the instructions of 8-bit operands add eight products at a time, each cut off
// 13 bits below the largest one's power of two. For codes of any size that is
// 2.9e-5 of the terms' magnitudes, and the sum of n terms of either sign is about
// sqrt(n) smaller than those: from 300 terms on more than float16's own rounding,
// 2^-11 of the result.
struct E4m3 {
  uint8_t bits;
};

// 16 codes times 2^(scale - 127) as bfloat16.
struct Wide {
  U32x4 v[2];
};
__device__ __forceinline__ Wide Widen(const U32x4& codes, int32_t scale) {
  const float s =
      __builtin_bit_cast(float, static_cast<uint32_t>(scale) << 23);
  Wide w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = codes[i];
    w.v[i / 2][i % 2 * 2] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, false));
    w.v[i / 2][i % 2 * 2 + 1] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, true));
  }
  return w;
}
// The exponents with which bfloat16 holds every code, 2^-9 to 448, as a normal
// value; of codes without a power of two.
constexpr int32_t kUnscaled = 127;
constexpr int32_t kLeastHeld = kUnscaled - 126 + 9;
constexpr int32_t kMostHeld = kUnscaled + 119;

// ---------------------------------------------------------------------------
// Rows in segments: those of expert e are [offsets[e], offsets[e + 1]); the
// ones behind the last and before the first belong to no expert.
// ---------------------------------------------------------------------------

// The rows of segment s, inside [0, n) whatever the offsets hold; segments
// `experts` and `experts` + 1 are the rows of none, behind and before.
constexpr int kNone = 2;
struct Segment {
  int32_t begin;
  int32_t end;
};
__device__ __forceinline__ Segment SegmentOf(const int32_t* offsets,
                                             int32_t experts, int32_t n,
                                             int32_t s) {
  if (s > experts) return {0, min(max(offsets[0], 0), n)};
  const int32_t begin = min(max(offsets[s], 0), n);
  const int32_t end = s < experts ? max(min(offsets[s + 1], n), begin) : n;
  return {begin, end};
}

// The rows [row, end) of the tile'th tile, and its segment (-1: no such tile).
// Every wavefront finds it by itself: a lane counts the tiles of neighbouring
// segments, the lanes' counts are added up.
struct RowTile {
  int32_t segment;
  int32_t row;
  int32_t end;
};
// Tiles of `rows` rows; the sum may pass 31 bits.
__device__ __forceinline__ int32_t TilesOf(const Segment& s, int32_t rows) {
  const uint32_t n = static_cast<uint32_t>(s.end - s.begin);
  return static_cast<int32_t>((n + static_cast<uint32_t>(rows) - 1) /
                              static_cast<uint32_t>(rows));
}
__device__ __forceinline__ RowTile FindRowTile(const int32_t* offsets,
                                               int32_t experts, int32_t n,
                                               int32_t tile, int32_t tile_rows) {
  // Without offsets all rows are the one expert's.
  if (offsets == nullptr) {
    if (tile >= (n + tile_rows - 1) / tile_rows) return {-1, 0, 0};
    return {0, tile * tile_rows, n};
  }
  // Segments of a lane.
  const int segments = experts + kNone;
  const int per = (segments + kWave - 1) / kWave;
  const int first = LaneId() * per;
  int32_t count = 0;
  for (int i = 0; i < per; ++i) {
    if (first + i < segments) {
      const Segment s = SegmentOf(offsets, experts, n, first + i);
      count += TilesOf(s, tile_rows);
    }
  }
  const int32_t upto = WaveInclusiveScan(count);
  const uint64_t past = __ballot(upto > tile);
  if (past == 0) return {-1, 0, 0};
  const int who = __builtin_ctzll(past);
  int32_t at = tile - __builtin_amdgcn_readlane(upto - count, who);
  for (int i = who * per;; ++i) {
    const Segment s = SegmentOf(offsets, experts, n, i);
    const int32_t tiles = TilesOf(s, tile_rows);
    if (at < tiles || i == segments - 1) {
      // Counts of segments that overlap may wrap: no tile then.
      if (at < 0 || at >= tiles) return {-1, 0, 0};
      return {__builtin_amdgcn_readfirstlane(i),
              __builtin_amdgcn_readfirstlane(s.begin + at * tile_rows),
              __builtin_amdgcn_readfirstlane(s.end)};
    }
    at -= tiles;
  }
}

// The number of tiles before segment `segment`; every wavefront by itself.
__device__ __forceinline__ int32_t TilesBefore(const int32_t* offsets,
                                               int32_t experts, int32_t n,
                                               int32_t segment,
                                               int32_t tile_rows) {
  int32_t count = 0;
  for (int s = LaneId(); s < segment; s += kWave) {
    count += TilesOf(SegmentOf(offsets, experts, n, s), tile_rows);
  }
  return __builtin_amdgcn_readlane(WaveInclusiveScan(count), kWave - 1);
}

// The expert with the `rank`th most rows (equal ones in their order); every
// wavefront by itself.
constexpr int kMostRanked = 4 * kWave;
__device__ __forceinline__ int32_t ExpertOfRank(const int32_t* offsets,
                                                int32_t experts, int32_t n,
                                                int32_t rank) {
  constexpr int kPer = kMostRanked / kWave;
  int32_t rows[kPer], before[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = i * kWave + LaneId();
    before[i] = 0;
    rows[i] = -1;
    if (e < experts) {
      const Segment s = SegmentOf(offsets, experts, n, e);
      rows[i] = s.end - s.begin;
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int some = min(experts - k * kWave, kWave);
    for (int j = 0; j < some; ++j) {
      const int32_t other = __builtin_amdgcn_readlane(rows[k], j);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        before[i] += other > rows[i] ||
                     (other == rows[i] && k * kWave + j < i * kWave + LaneId());
      }
    }
  }
  int32_t found = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint64_t here =
        __ballot(before[i] == rank && i * kWave + LaneId() < experts);
    if (here != 0) found = i * kWave + __builtin_ctzll(here);
  }
  return __builtin_amdgcn_readfirstlane(found);
}

// Tiles of a matrix in the order of the work-groups. Work-groups go to the
// eight XCDs in turn; each XCD gets patches of up to `most` tiles that share
// operands in its L2, 32 being one for each of its CUs.
struct TileGrid {
  static constexpr int32_t kMost = 1 << 30;
  int32_t rows;     // tiles
  int32_t columns;
  int32_t patch_rows;
  int32_t patch_columns;

  // More than a launch takes are cut: Groups() says so then.
  TileGrid(int64_t r, int64_t c, int64_t most = 32)
      : rows(static_cast<int32_t>(r < kMost ? r : kMost)),
        columns(static_cast<int32_t>(c < kMost ? c : kMost)) {
    const int32_t size = static_cast<int32_t>(most < 1 ? 1 : most);
    const int32_t wide = size >= 32 ? 8 : size >= 8 ? 4 : size >= 2 ? 2 : 1;
    patch_columns = columns < wide ? columns : wide;
    patch_rows = size / patch_columns;
    if (patch_rows > rows) patch_rows = rows;
  }
  int64_t Groups() const {
    const int64_t patches =
        CeilDiv(rows, patch_rows) * CeilDiv(columns, patch_columns);
    return RoundUp(patches, 8) * patch_rows * patch_columns;
  }
  // False: no such tile.
  __device__ __forceinline__ bool Tile(uint32_t group, int32_t* row,
                                       int32_t* column) const {
    const uint32_t size = patch_rows * patch_columns;
    const uint32_t xcd = group % 8, within = group / 8 % size;
    const uint32_t patch = group / 8 / size * 8 + xcd;
    const uint32_t across = (columns + patch_columns - 1) / patch_columns;
    *row = patch / across * patch_rows + within % patch_rows;
    *column = patch % across * patch_columns + within / patch_rows;
    return *row < rows && *column < columns;
  }
};

// ---------------------------------------------------------------------------
// Results.
// ---------------------------------------------------------------------------

// Elements [column, column + V) of a row, those below `columns`.
template <typename T, int V>
__device__ __forceinline__ void StoreUpTo(T* row, int32_t column,
                                          int32_t columns,
                                          const Vec<T, V>& x) {
  if (column + V <= columns) {
    StoreVec<T, V>(row + column, x);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (column + j < columns) row[column + j] = x.v[j];
    }
  }
}

// 32 rows of kFragments * 32 columns from their accumulators, rounded once. A
// lane's values are spread over its row: they go through `lds` (the wavefront's
// own) and leave as whole rows, neighbouring lanes writing
// neighbouring 16 bytes. c is the first row's first element of the tile's
// matrix of `columns` columns, of which `n` are left, and `m` rows.
template <typename T, int kFragments>
struct RowsOut {
  static constexpr int kRowBytes = kFragments * 32 * sizeof(T);
  static constexpr int kBytes = 32 * kRowBytes;
  static constexpr int kChunks = kRowBytes / 16;
  static_assert(kChunks == 4 || kChunks == 8 || kChunks == 16, "row of a lane");

  // 16 lanes that access one chunk of 16 rows find them in different banks.
  static __device__ __forceinline__ int Key(int row) {
    return row / (16 / kChunks) % kChunks;
  }
  static __device__ __forceinline__ void Store(const F32x16* acc, char* lds,
                                               T* c, int64_t columns, int m,
                                               int n) {
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x % kWave;
    const int row = lane % 32, h = lane / 32;
#pragma unroll
    for (int f = 0; f < kFragments; ++f) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        Vec<T, 4> v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.v[i] = static_cast<T>(acc[f][q * 4 + i]);
        const int at = f * 32 + q * 8 + h * 4;  // its column
        char* p = lds + row * kRowBytes + ((at / V) ^ Key(row)) * 16 +
                  at % V * sizeof(T);
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<U32x4*>(p) = __builtin_bit_cast(U32x4, v);
        } else {
          *reinterpret_cast<uint2*>(p) = __builtin_bit_cast(uint2, v);
        }
      }
    }
    constexpr int kAtOnce = kWave / kChunks;  // rows
#pragma unroll
    for (int i = 0; i < 32 / kAtOnce; ++i) {
      const int r = i * kAtOnce + lane / kChunks, chunk = lane % kChunks;
      const U32x4 x = *reinterpret_cast<const U32x4*>(
          lds + r * kRowBytes + (chunk ^ Key(r)) * 16);
      if (r < m) {
        StoreUpTo(c + r * columns, chunk * V, n,
                  __builtin_bit_cast(Vec<T, V>, x));
      }
    }
  }
};

// ---------------------------------------------------------------------------
// A tile of the result by one work-group of kWavesM x kWavesN wavefronts. Of
// two steps of the depth in LDS one is multiplied while the other is loaded.
// ---------------------------------------------------------------------------

template <typename T_, Along kA, Along kB, int kM_, int kN_, int kWavesM,
          int kWavesN, bool kDirect_>
struct Tile {
  using T = T_;
  static constexpr int kM = kM_, kN = kN_;
  static constexpr int kWaves = kWavesM * kWavesN;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr bool kDirect = kDirect_;
  static constexpr int kFragM = kM / kWavesM / 32;
  static constexpr int kFragN = kN / kWavesN / 32;
  using A = Panel<T, kA, kM, kThreads>;
  using B = Panel<T, kB, kN, kThreads>;
  static constexpr int kDepth = A::kDepth;
  static constexpr int kLds = A::kBytes + B::kBytes;
  static constexpr Along kAlongA = kA, kAlongB = kB;

  F32x16 acc[kFragM][kFragN];

  static __device__ __forceinline__ int WaveM() {
    return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) / kWavesN *
           (kFragM * 32);
  }
  static __device__ __forceinline__ int WaveN() {
    return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) % kWavesN *
           (kFragN * 32);
  }

  // What half a step is multiplied from.
  struct Fragments {
    U32x4 a[2][kFragM];
    U32x4 b[2][kFragN];
  };
  static __device__ __forceinline__ void Read(const char* lds, int half,
                                              Fragments* f) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < kFragN; ++j) {
        f->b[q][j] =
            B::Fragment(lds, A::kBytes, WaveN() + j * 32, half * 2 + q);
      }
#pragma unroll
      for (int i = 0; i < kFragM; ++i) {
        f->a[q][i] = A::Fragment(lds, 0, WaveM() + i * 32, half * 2 + q);
      }
    }
  }
  template <typename Scales>
  __device__ __forceinline__ void Multiply(const Fragments& f,
                                           const Scales& scales) {
    if constexpr (sizeof(T) == 1) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        Wide b[kFragN];
#pragma unroll
        for (int j = 0; j < kFragN; ++j) b[j] = Widen(f.b[q][j], scales.b);
#pragma unroll
        for (int i = 0; i < kFragM; ++i) {
          const Wide a = Widen(f.a[q][i], scales.a[i]);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int j = 0; j < kFragN; ++j) {
              MultiplyAdd<bf16>(b[j].v[part], a.v[part], &acc[i][j]);
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int i = 0; i < kFragM; ++i) {
#pragma unroll
          for (int j = 0; j < kFragN; ++j) {
            MultiplyAdd<T>(f.b[q][j], f.a[q][i], &acc[i][j]);
          }
        }
      }
    }
  }

  // The products so far are made here: without side effects, the compiler moves
  // them behind barriers and the reads that follow.
  __device__ __forceinline__ void Stay() {
#pragma unroll
    for (int i = 0; i < kFragM; ++i) {
#pragma unroll
      for (int j = 0; j < kFragN; ++j) asm volatile("" : "+v"(acc[i][j]));
    }
  }

  // The tile's sums over `depth`. a and b are the panels' first elements; m and
  // n (at least 1) the outer indices that exist; the totals the elements of a row
  // of the operands in memory. lds0 and lds1 are different
  // arrays: the compiler has to see that a load into one needs no wait before
  // the other is read. scales: those of 8-bit operands, which are loaded a step
  // ahead as the operands are.
  template <typename Scales>
  __device__ __forceinline__ void Run(const T* a, int64_t a_stride, int m,
                                      int32_t a_total, const T* b,
                                      int64_t b_stride, int n,
                                      int32_t b_total, int32_t depth,
                                      char* lds0, char* lds1,
                                      Scales&& scales) {
#pragma unroll
    for (int i = 0; i < kFragM; ++i) {
#pragma unroll
      for (int j = 0; j < kFragN; ++j) acc[i][j] = F32x16{};
    }
    if (depth <= 0) return;
    const int64_t a_step =
        kA == Along::kDepth ? kDepth : kDepth * a_stride;
    const int64_t b_step =
        kB == Along::kDepth ? kDepth : kDepth * b_stride;
    if constexpr (kDirect) {
      A pa;
      B pb;
      pa.Start(a_stride, m);
      pb.Start(b_stride, n);
      const char* at_a = reinterpret_cast<const char*>(a);
      const char* at_b = reinterpret_cast<const char*>(b);
      const auto load = [&](char* lds) __attribute__((always_inline)) {
        pa.Load(at_a, lds);
        pb.Load(at_b, lds + A::kBytes);
        at_a += a_step * sizeof(T);
        at_b += b_step * sizeof(T);
      };
      // What is no whole step comes first, through registers (8 bits have no
      // such steps).
      int32_t left = sizeof(T) == 1 ? 0 : depth % kDepth;
      if (left != 0) {
        typename A::Chunks ca;
        typename B::Chunks cb;
        A::template Fetch<true>(a, a_stride, m, left, 0, &ca);
        B::template Fetch<true>(b, b_stride, n, left, 0, &cb);
        A::Put(ca, lds0);
        B::Put(cb, lds0 + A::kBytes);
        at_a += a_step / kDepth * left * sizeof(T);
        at_b += b_step / kDepth * left * sizeof(T);
      } else {
        left = kDepth;
        load(lds0);
        scales.Load();
      }
      int32_t ahead = (depth - left) / kDepth;  // steps behind the current one
      WaitLoads<0>();
      Barrier();
      // With two wavefronts a SIMD one reads while the other multiplies: the
      // second half of them are a barrier behind.
      constexpr bool kTurns = kWaves == 8;
      const bool second =
          __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) >= kWaves / 2;
      if (kTurns && second) Barrier();
      const auto half = [&](const char* now, int h) __attribute__((
                            always_inline)) {
        Fragments f;
        Read(now, h, &f);
        if constexpr (kTurns) {
          // Whoever reads the next step first has its loads waited for by all.
          if (h == 1) WaitLoads<0>();
          Barrier();
          __builtin_amdgcn_s_setprio(1);
          Multiply(f, scales);
          Stay();
          __builtin_amdgcn_s_setprio(0);
          Barrier();
        } else {
          __builtin_amdgcn_sched_barrier(0);
          Multiply(f, scales);
          Stay();
          __builtin_amdgcn_sched_barrier(0);
          if (h == 1) {
            WaitLoads<0>();
            Barrier();
          }
        }
      };
      const auto turn = [&](const char* now, char* next) __attribute__((
                            always_inline)) {
        scales.Take();
        if (ahead > 0) {
          load(next);
          scales.Load();
        }
        half(now, 0);
        half(now, 1);
        --ahead;
      };
      while (ahead >= 1) {
        turn(lds0, lds1);
        turn(lds1, lds0);
      }
      if (ahead == 0) turn(lds0, lds1);
      if (kTurns && !second) Barrier();
    } else {
      typename A::Chunks ca;
      typename B::Chunks cb;
      A::template Fetch<false>(a, a_stride, m, depth, a_total, &ca);
      B::template Fetch<false>(b, b_stride, n, depth, b_total, &cb);
      for (int32_t at = 0; at < depth; at += kDepth) {
        char* lds = (at / kDepth & 1) ? lds1 : lds0;
        A::Put(ca, lds);
        B::Put(cb, lds + A::kBytes);
        __syncthreads();
        a += a_step;
        b += b_step;
        if (at + kDepth < depth) {
          const int32_t rest = depth - at - kDepth;
          A::template Fetch<false>(a, a_stride, m, rest, a_total, &ca);
          B::template Fetch<false>(b, b_stride, n, rest, b_total, &cb);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Fragments f;
          Read(lds, h, &f);
          Multiply(f, scales);
        }
      }
      __syncthreads();
    }
  }

  // Stores what exists of the tile: c is its first element, m and n the rows
  // and columns from there on.
  template <typename Out>
  __device__ __forceinline__ void Store(Out* c, int64_t stride, int m, int n,
                                        char* lds) const {
    using R = RowsOut<Out, kFragN>;
    static_assert(R::kBytes * kWaves <= kLds, "every wavefront its own");
    lds += __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * R::kBytes;
#pragma unroll
    for (int i = 0; i < kFragM; ++i) {
      const int row = WaveM() + i * 32;
      R::Store(acc[i], lds, c + row * stride + WaveN(), stride, m - row,
               n - WaveN());
    }
  }
};

// No scales: operands of 16 or 32 bits.
struct NoScales {
  __device__ __forceinline__ void Load() {}
  __device__ __forceinline__ void Take() {}
};

// The work-group sizes of a product, and its kinds of tiles: for few rows of an
// expert, for most calls, and for many.
template <typename T, Along kA, Along kB, bool kDirect>
using SmallTile = Tile<T, kA, kB, 32, 128, 1, 4, kDirect>;
template <typename T, Along kA, Along kB, bool kDirect>
using MiddleTile = Tile<T, kA, kB, 128, 128, 2, 2, kDirect>;
template <typename T, Along kA, Along kB>
using LargeTile = Tile<T, kA, kB, 256, 256, 2, 4, true>;

constexpr int kCus = 256;

// Whether small tiles are worth it: rows of an expert are few, or middle ones
// would leave a quarter of the CUs without work (float32, 1000 rows of 4 experts,
// 2048 x 256, 16 tiles: 141 us, 53 with small ones; bfloat16, 2000 rows, 1024 x
// 1024, 128 tiles: 16 and 11; 3900 rows, 248 tiles: 16 and 18).
inline bool WorthSmall(int64_t rows, int64_t columns, int64_t experts) {
  return rows <= 32 * experts ||
         4 * CeilDiv(rows, 128) * CeilDiv(columns, 128) < 3 * kCus;
}

// Whether large tiles, one at a time on a CU, are worth it: they are up to a fifth
// faster where the last round of them is full enough (64 experts, 131,072 rows,
// 1024 x 4096: bfloat16 1173 us, with middle ones 1417; 8 bits 1200 and 1283 on one
// box; but 20,011 rows, 3328 x 1000, which is 316 tiles, 8 bits 194 and 148).
inline bool WorthLarge(int64_t rows, int64_t columns) {
  const int64_t tiles = CeilDiv(rows, 256) * CeilDiv(columns, 256);
  return 5 * tiles >= 4 * RoundUp(tiles, kCus);
}

}  // namespace scemb
