// Tokens ordered by expert and back: a stable counting sort of the choices,
// the copy of the tokens' rows to their places, the weighted sum of the rows
// back at their tokens, and the gradients.
//
// The sort knows both where a choice goes (positions) and where it came from
// (sources), so every kernel works token by token: it reads a token's row
// once however many choices it has, writes whole rows, and sums in the order
// of the choices. Nothing is added atomically.
#include <algorithm>

#include "dense.h"

namespace scemb {
namespace {

// ---------------------------------------------------------------------------
// Counting sort.
// ---------------------------------------------------------------------------

constexpr int kTileWaves = 4;        // work-group of a tile
constexpr int kSingleWaves = 16;     // work-group of a sort in one launch
constexpr int64_t kTile = 2048;      // ids of a tile, or a multiple of it
constexpr int64_t kMaxTiles = 2048;  // counts of all tiles are scanned
// Up to here one work-group sorts by itself, in one launch instead of three
// (where its counts fit 64 KB of LDS).
constexpr int64_t kSingle = 8192;
constexpr int kKeyBits = 11;  // 0..SCEMB_MAX_EXPERTS
static_assert(SCEMB_MAX_EXPERTS < (1 << kKeyBits), "keys of kKeyBits bits");

// The expert of choice i, `experts` for a dropped one.
template <typename I>
__device__ __forceinline__ uint32_t KeyOf(const I* ids, int64_t i,
                                          int32_t experts) {
  const I id = ids[i];
  return id >= 0 && id < static_cast<I>(experts) ? static_cast<uint32_t>(id)
                                                 : experts;
}

// Counts the keys of each wavefront's share [first, last) of a tile into its
// row of `counts` ([waves][experts + 1] in LDS, cleared here).
template <typename I, int kWaves>
__device__ __forceinline__ void CountShares(const I* ids, int32_t experts,
                                            int64_t first, int64_t last,
                                            uint32_t* counts) {
  const int row = experts + 1;
  for (int i = threadIdx.x; i < kWaves * row; i += kWaves * kWave) {
    counts[i] = 0;
  }
  __syncthreads();
  uint32_t* mine = counts + (threadIdx.x / kWave) * row;
  for (int64_t i = first + threadIdx.x % kWave; i < last; i += kWave) {
    atomicAdd(&mine[KeyOf(ids, i, experts)], 1u);
  }
  __syncthreads();
}

// Places a wavefront's share: next[key] is the place of its next choice of
// that key. 64 choices at a time, equal keys ranked by lane.
template <typename I>
__device__ __forceinline__ void PlaceShare(const I* ids, int32_t experts,
                                           int64_t first, int64_t last,
                                           uint32_t* next, int32_t* positions,
                                           int32_t* sources) {
  const int lane = threadIdx.x % kWave;
  for (int64_t at = first; at < last; at += kWave) {
    const int64_t i = at + lane;
    const bool in = i < last;
    const uint32_t key = in ? KeyOf(ids, i, experts) : 0u;
    const uint64_t same = MatchLanes<kKeyBits>(__ballot(in), key);
    const int leader = in ? __ffsll(static_cast<unsigned long long>(same)) - 1
                          : lane;
    uint32_t base = 0;
    if (in && lane == leader) {
      base = atomicAdd(&next[key], static_cast<uint32_t>(__popcll(same)));
    }
    base = __shfl(base, leader, kWave);
    if (in) {
      const uint32_t place = base + __popcll(same & LaneMaskLt());
      positions[i] = static_cast<int32_t>(place);
      sources[place] = static_cast<int32_t>(i);
    }
  }
}

struct Share {
  int64_t first;
  int64_t last;
};
// The wavefront's share of ids [begin, end): whole steps of 64.
template <int kWaves>
__device__ __forceinline__ Share ShareOf(int64_t begin, int64_t end) {
  const int64_t steps = (end - begin + kWave - 1) / kWave;
  const int64_t per = (steps + kWaves - 1) / kWaves * kWave;
  const int64_t first = begin + per * (threadIdx.x / kWave);
  return {first < end ? first : end, first + per < end ? first + per : end};
}

// One work-group sorts everything.
template <typename I>
__global__ __launch_bounds__(kSingleWaves* kWave) void SortSingle(
    const I* ids, int64_t n, int32_t experts, int32_t* positions,
    int32_t* sources, int32_t* offsets) {
  constexpr int kBlock = kSingleWaves * kWave;
  static_assert(SCEMB_MAX_EXPERTS <= kBlock, "an expert a thread");
  extern __shared__ uint32_t counts[];
  __shared__ uint32_t scan[kSingleWaves + 1];
  const int row = experts + 1;
  const Share s = ShareOf<kSingleWaves>(0, n);
  CountShares<I, kSingleWaves>(ids, experts, s.first, s.last, counts);
  const int e = threadIdx.x;
  uint32_t mine = 0;
  if (e < experts) {
    for (int w = 0; w < kSingleWaves; ++w) mine += counts[w * row + e];
  }
  uint32_t kept = 0;
  uint32_t place = BlockExclusiveScan<uint32_t, kBlock>(mine, scan, &kept);
  if (e < experts) {
    offsets[e] = static_cast<int32_t>(place);
    for (int w = 0; w < kSingleWaves; ++w) {
      const uint32_t c = counts[w * row + e];
      counts[w * row + e] = place;
      place += c;
    }
  }
  if (e == 0) {
    offsets[experts] = static_cast<int32_t>(kept);
    uint32_t dropped = kept;
    for (int w = 0; w < kSingleWaves; ++w) {
      const uint32_t c = counts[w * row + experts];
      counts[w * row + experts] = dropped;
      dropped += c;
    }
  }
  __syncthreads();
  PlaceShare(ids, experts, s.first, s.last,
             counts + (threadIdx.x / kWave) * row, positions, sources);
}

// Counts of each tile: hist[key][tile].
template <typename I>
__global__ __launch_bounds__(kTileWaves* kWave) void CountTiles(
    const I* ids, int64_t n, int32_t experts, int64_t tile, uint32_t* hist) {
  constexpr int kBlock = kTileWaves * kWave;
  extern __shared__ uint32_t counts[];
  const int row = experts + 1;
  for (int i = threadIdx.x; i < row; i += kBlock) counts[i] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * tile;
  const int64_t end = begin + tile < n ? begin + tile : n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kBlock) {
    atomicAdd(&counts[KeyOf(ids, i, experts)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < row; i += kBlock) {
    hist[static_cast<int64_t>(i) * gridDim.x + blockIdx.x] = counts[i];
  }
}

// Exclusive sums of each key's counts over the tiles, in place, and their
// total. A wavefront a key.
__global__ __launch_bounds__(256) void ScanTiles(uint32_t* hist, int32_t tiles,
                                                 int32_t keys,
                                                 uint32_t* totals) {
  const int key = blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  if (key >= keys) return;
  const int lane = threadIdx.x % kWave;
  uint32_t* mine = hist + static_cast<int64_t>(key) * tiles;
  uint32_t run = 0;
  for (int at = 0; at < tiles; at += kWave) {
    const int i = at + lane;
    const uint32_t c = i < tiles ? mine[i] : 0u;
    const uint32_t inc = WaveInclusiveScan(c);
    if (i < tiles) mine[i] = run + inc - c;
    run += __shfl(inc, kWave - 1, kWave);
  }
  if (lane == 0) totals[key] = run;
}

// Places each tile's choices. Every work-group sums the keys' totals itself.
template <typename I>
__global__ __launch_bounds__(kTileWaves* kWave) void PlaceTiles(
    const I* ids, int64_t n, int32_t experts, int64_t tile,
    const uint32_t* hist, const uint32_t* totals, int32_t* positions,
    int32_t* sources, int32_t* offsets) {
  constexpr int kBlock = kTileWaves * kWave;
  extern __shared__ uint32_t counts[];
  __shared__ uint32_t scan[kTileWaves + 1];
  const int row = experts + 1;
  const int64_t begin = blockIdx.x * tile;
  const int64_t end = begin + tile < n ? begin + tile : n;
  const Share s = ShareOf<kTileWaves>(begin, end);
  CountShares<I, kTileWaves>(ids, experts, s.first, s.last, counts);
  uint32_t run = 0;
  for (int at = 0; at < row; at += kBlock) {
    const int e = at + threadIdx.x;
    const uint32_t total = e < row ? totals[e] : 0u;
    uint32_t sum = 0;
    const uint32_t before =
        run + BlockExclusiveScan<uint32_t, kBlock>(total, scan, &sum);
    run += sum;
    if (e < row) {
      if (blockIdx.x == 0) offsets[e] = static_cast<int32_t>(before);
      uint32_t place =
          before + hist[static_cast<int64_t>(e) * gridDim.x + blockIdx.x];
      for (int w = 0; w < kTileWaves; ++w) {
        const uint32_t c = counts[w * row + e];
        counts[w * row + e] = place;
        place += c;
      }
    }
  }
  __syncthreads();
  PlaceShare(ids, experts, s.first, s.last,
             counts + (threadIdx.x / kWave) * row, positions, sources);
}

// Ids of a tile and their number: at least one of each, as the offsets of no
// choices are written too.
int64_t TileOf(int64_t n) {
  return kTile * CeilDiv(std::max<int64_t>(n, 1), kTile * kMaxTiles);
}
int64_t TilesOf(int64_t n) {
  return CeilDiv(std::max<int64_t>(n, 1), TileOf(n));
}

bool SortsSingle(int64_t n, int32_t experts) {
  return n <= kSingle &&
         sizeof(uint32_t) * kSingleWaves * (experts + 1) <= 65536 - 256;
}

template <typename I>
int Sort(const void* ids, int64_t n, int32_t experts, int32_t* positions,
         int32_t* sources, int32_t* offsets, void* workspace,
         size_t workspace_bytes, hipStream_t stream) {
  const I* in = static_cast<const I*>(ids);
  const size_t row = sizeof(uint32_t) * (experts + 1);
  if (SortsSingle(n, experts)) {
    hipLaunchKernelGGL(SortSingle<I>, dim3(1), dim3(kSingleWaves * kWave),
                       kSingleWaves * row, stream, in, n, experts, positions,
                       sources, offsets);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }
  const int64_t tile = TileOf(n);
  const uint32_t tiles = static_cast<uint32_t>(TilesOf(n));
  Arena arena(workspace, workspace_bytes);
  uint32_t* hist = arena.Take<uint32_t>((experts + 1) *
                                        static_cast<int64_t>(tiles));
  uint32_t* totals = arena.Take<uint32_t>(experts + 1);
  if (workspace == nullptr || arena.overflow()) {
    return Fail(SCEMB_ERR_WORKSPACE,
                "sort by expert: workspace missing or too small");
  }
  hipLaunchKernelGGL(CountTiles<I>, dim3(tiles), dim3(kTileWaves * kWave), row,
                     stream, in, n, experts, tile, hist);
  SCEMB_LAUNCH_CHECK();
  hipLaunchKernelGGL(ScanTiles, dim3((experts + 4) / 4), dim3(256), 0, stream,
                     hist, static_cast<int32_t>(tiles), experts + 1, totals);
  SCEMB_LAUNCH_CHECK();
  hipLaunchKernelGGL(PlaceTiles<I>, dim3(tiles), dim3(kTileWaves * kWave),
                     kTileWaves * row, stream, in, n, experts, tile, hist,
                     totals, positions, sources, offsets);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

// ---------------------------------------------------------------------------
// Rows to their experts and back. G neighbouring lanes have a token.
// ---------------------------------------------------------------------------

constexpr int kRowBlock = 256;

struct Order {
  const int32_t* positions;
  const int32_t* kept;  // offsets[num_experts]
  int64_t tokens;
  int32_t choices;

  // Choices that are kept, at most as many as there are.
  __device__ __forceinline__ uint32_t Kept() const {
    const int64_t n = tokens * choices;
    const int64_t k = *kept;
    return static_cast<uint32_t>(k < n ? k : n);
  }
};

// U: an unsigned type that row starts and the row's length are multiples of.
template <typename U, int G>
__global__ __launch_bounds__(kRowBlock) void ToExperts(const U* x,
                                                       int64_t stride,
                                                       int32_t units,
                                                       Order order, U* rows) {
  constexpr int kTokens = kRowBlock / G;
  const int lane = threadIdx.x % G;
  const uint32_t kept = order.Kept();
  const uint32_t all = static_cast<uint32_t>(order.tokens * order.choices);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens +
                   threadIdx.x / G;
       t < order.tokens; t += static_cast<int64_t>(gridDim.x) * kTokens) {
    const int32_t* places = order.positions + t * order.choices;
    for (int32_t c = lane; c < units; c += G) {
      const U v = x[t * stride + c];
      for (int k = 0; k < order.choices; ++k) {
        const uint32_t p = static_cast<uint32_t>(places[k]);
        if (p < all) {
          rows[static_cast<int64_t>(p) * units + c] = p < kept ? v : U{};
        }
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float WeightAt(const void* w, bool f32, int64_t i) {
  return w == nullptr ? 1.f
         : f32        ? static_cast<const float*>(w)[i]
                      : static_cast<float>(static_cast<const T*>(w)[i]);
}

template <typename T, int V, int G>
__global__ __launch_bounds__(kRowBlock) void FromExperts(
    const T* rows, int64_t stride, int32_t dim, const void* weights,
    bool weights_f32, Order order, T* y) {
  constexpr int kTokens = kRowBlock / G;
  const int lane = threadIdx.x % G;
  const uint32_t kept = order.Kept();
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens +
                   threadIdx.x / G;
       t < order.tokens; t += static_cast<int64_t>(gridDim.x) * kTokens) {
    const int64_t first = t * order.choices;
    for (int32_t c = lane * V; c < dim; c += G * V) {
      float sum[V];
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.f;
#pragma unroll 2
      for (int k = 0; k < order.choices; ++k) {
        const uint32_t p = static_cast<uint32_t>(order.positions[first + k]);
        if (p < kept) {
          const float w = WeightAt<T>(weights, weights_f32, first + k);
          const auto v = LoadVec<T, V>(rows + p * stride + c);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            sum[j] = fmaf(w, static_cast<float>(v.v[j]), sum[j]);
          }
        }
      }
      Vec<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) out.v[j] = static_cast<T>(sum[j]);
      StoreVec<T, V>(y + t * dim + c, out);
    }
  }
}

template <typename T, int V, int G>
__global__ __launch_bounds__(kRowBlock) void FromExpertsGrad(
    const T* dy, int64_t dy_stride, const T* rows, int64_t stride, int32_t dim,
    const void* weights, bool weights_f32, Order order, T* drows,
    void* dweights) {
  constexpr int kTokens = kRowBlock / G;
  const int lane = threadIdx.x % G;
  const uint32_t kept = order.Kept();
  const uint32_t all = static_cast<uint32_t>(order.tokens * order.choices);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens +
                   threadIdx.x / G;
       t < order.tokens; t += static_cast<int64_t>(gridDim.x) * kTokens) {
    for (int k = 0; k < order.choices; ++k) {
      const int64_t at = t * order.choices + k;
      const uint32_t p = static_cast<uint32_t>(order.positions[at]);
      const bool keep = p < kept;
      const float w = keep ? WeightAt<T>(weights, weights_f32, at) : 0.f;
      float dot = 0.f;
      if (p < all) {
        for (int32_t c = lane * V; c < dim; c += G * V) {
          Vec<T, V> out;
          if (keep) {
            const auto g = LoadVec<T, V>(dy + t * dy_stride + c);
            const auto v = LoadVec<T, V>(rows + p * stride + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float gj = static_cast<float>(g.v[j]);
              dot = fmaf(gj, static_cast<float>(v.v[j]), dot);
              out.v[j] = static_cast<T>(w * gj);
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = static_cast<T>(0.f);
          }
          StoreVec<T, V>(drows + static_cast<int64_t>(p) * dim + c, out);
        }
      }
      dot = LaneSum<G>(dot);
      if (lane == 0 && dweights != nullptr) {
        if (weights_f32) {
          static_cast<float*>(dweights)[at] = dot;
        } else {
          static_cast<T*>(dweights)[at] = static_cast<T>(dot);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

uint32_t RowGrid(int64_t tokens, int g) {
  return static_cast<uint32_t>(
      std::min<int64_t>(CeilDiv(tokens, kRowBlock / g), 0x7fffffff));
}

Order OrderOf(const scemb_expert_order_t* o) {
  return {o->positions, o->offsets + o->num_experts, o->tokens, o->choices};
}

int CheckOrder(const scemb_expert_order_t* o, int32_t type, int64_t dim) {
  if (o == nullptr || TypeBytes(type) == 0) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "experts: the order is missing, or rows are not float32, "
                "bfloat16 or float16");
  }
  if (dim < 1 || dim > 0x7fffffff - 65536 || o->tokens < 0 ||
      o->choices < 1 || o->num_experts < 1 ||
      o->num_experts > SCEMB_MAX_EXPERTS ||
      o->tokens > 0x7fffffff / o->choices) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "experts: dim outside [1, 2^31 - 2^16), tokens below 0, "
                "choices below 1, more than 2^31 - 1 choices in all, or "
                "experts outside [1, 1024]");
  }
  if (o->tokens > 0 && (o->positions == nullptr || o->offsets == nullptr)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "experts: positions or offsets missing");
  }
  return 0;
}

template <typename U>
int RunToExperts(const void* x, int64_t stride_bytes, int64_t row_bytes,
                 const Order& o, void* rows, hipStream_t stream) {
  const int32_t units = static_cast<int32_t>(row_bytes / sizeof(U));
  const int64_t stride = stride_bytes / static_cast<int64_t>(sizeof(U));
  const U* src = static_cast<const U*>(x);
  U* dst = static_cast<U*>(rows);
  if (units <= 16) {
    hipLaunchKernelGGL((ToExperts<U, 16>), dim3(RowGrid(o.tokens, 16)),
                       dim3(kRowBlock), 0, stream, src, stride, units, o, dst);
  } else {
    hipLaunchKernelGGL((ToExperts<U, 64>), dim3(RowGrid(o.tokens, 64)),
                       dim3(kRowBlock), 0, stream, src, stride, units, o, dst);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T, int V>
int RunFromExperts(const T* rows, int64_t stride, int64_t dim,
                   const void* weights, bool f32, const Order& o, T* y,
                   hipStream_t stream) {
  const int32_t d = static_cast<int32_t>(dim);
  if (dim <= 16 * V) {
    hipLaunchKernelGGL((FromExperts<T, V, 16>), dim3(RowGrid(o.tokens, 16)),
                       dim3(kRowBlock), 0, stream, rows, stride, d, weights,
                       f32, o, y);
  } else {
    hipLaunchKernelGGL((FromExperts<T, V, 64>), dim3(RowGrid(o.tokens, 64)),
                       dim3(kRowBlock), 0, stream, rows, stride, d, weights,
                       f32, o, y);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int FromExpertsOf(const void* rows, int64_t stride, int64_t dim,
                  const void* weights, bool f32, const Order& o, void* y,
                  hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const T* r = static_cast<const T*>(rows);
  T* out = static_cast<T*>(y);
  if (dim % V == 0 && stride % V == 0 && AlignedTo(rows, 16) &&
      AlignedTo(y, 16)) {
    return RunFromExperts<T, V>(r, stride, dim, weights, f32, o, out, stream);
  }
  return RunFromExperts<T, 1>(r, stride, dim, weights, f32, o, out, stream);
}

template <typename T, int V>
int RunFromExpertsGrad(const T* dy, int64_t dy_stride, const T* rows,
                       int64_t stride, int64_t dim, const void* weights,
                       bool f32, const Order& o, T* drows, void* dweights,
                       hipStream_t stream) {
  const int32_t d = static_cast<int32_t>(dim);
  if (dim <= 16 * V) {
    hipLaunchKernelGGL((FromExpertsGrad<T, V, 16>),
                       dim3(RowGrid(o.tokens, 16)), dim3(kRowBlock), 0, stream,
                       dy, dy_stride, rows, stride, d, weights, f32, o, drows,
                       dweights);
  } else {
    hipLaunchKernelGGL((FromExpertsGrad<T, V, 64>),
                       dim3(RowGrid(o.tokens, 64)), dim3(kRowBlock), 0, stream,
                       dy, dy_stride, rows, stride, d, weights, f32, o, drows,
                       dweights);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int FromExpertsGradOf(const void* dy, int64_t dy_stride, const void* rows,
                      int64_t stride, int64_t dim, const void* weights,
                      bool f32, const Order& o, void* drows, void* dweights,
                      hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const T* g = static_cast<const T*>(dy);
  const T* r = static_cast<const T*>(rows);
  T* out = static_cast<T*>(drows);
  if (dim % V == 0 && stride % V == 0 && dy_stride % V == 0 &&
      AlignedTo(dy, 16) && AlignedTo(rows, 16) && AlignedTo(drows, 16)) {
    return RunFromExpertsGrad<T, V>(g, dy_stride, r, stride, dim, weights, f32,
                                    o, out, dweights, stream);
  }
  return RunFromExpertsGrad<T, 1>(g, dy_stride, r, stride, dim, weights, f32, o,
                                  out, dweights, stream);
}

}  // namespace
}  // namespace scemb

extern "C" {

size_t scemb_sort_by_expert_workspace_size(int64_t n, int32_t num_experts) {
  using namespace scemb;
  if (n < 0 || n > 0x7fffffff || num_experts < 1 ||
      num_experts > SCEMB_MAX_EXPERTS) {
    SetError("sort by expert: choices or experts out of range");
    return 0;
  }
  Arena arena(nullptr, 0);
  if (!SortsSingle(n, num_experts)) {
    arena.Take<uint32_t>((num_experts + 1) * TilesOf(n));
  }
  arena.Take<uint32_t>(num_experts + 1);
  return arena.used();
}

int scemb_sort_by_expert(const void* ids, int32_t id_bytes, int64_t n,
                         int32_t num_experts, int32_t* positions,
                         int32_t* sources, int32_t* offsets, void* workspace,
                         size_t workspace_bytes, void* stream) {
  using namespace scemb;
  if (n < 0 || n > 0x7fffffff || num_experts < 1 ||
      num_experts > SCEMB_MAX_EXPERTS || (id_bytes != 4 && id_bytes != 8)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "sort by expert: ids are int32 or int64, at most 2^31 - 1 of "
                "them, experts within [1, 1024]");
  }
  if (offsets == nullptr || (n > 0 && (ids == nullptr || positions == nullptr ||
                                       sources == nullptr))) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "sort by expert: an operand is missing");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return id_bytes == 4
             ? Sort<int32_t>(ids, n, num_experts, positions, sources, offsets,
                             workspace, workspace_bytes, s)
             : Sort<int64_t>(ids, n, num_experts, positions, sources, offsets,
                             workspace, workspace_bytes, s);
}

int scemb_tokens_to_experts(const void* x, int32_t type, int64_t x_stride,
                            int64_t dim, const scemb_expert_order_t* order,
                            void* rows, void* stream) {
  using namespace scemb;
  const int bad = CheckOrder(order, type, dim);
  if (bad != 0) return bad;
  if (order->tokens == 0) return SCEMB_OK;
  if (x == nullptr || rows == nullptr || x_stride < 0) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "tokens to experts: x or rows missing, or a negative stride");
  }
  const Order o = OrderOf(order);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row = dim * TypeBytes(type);
  const int64_t stride = x_stride * TypeBytes(type);
  // The widest unit that divides all row starts: bytes are only moved.
  const uint64_t bits = static_cast<uint64_t>(row) |
                        static_cast<uint64_t>(stride) |
                        reinterpret_cast<uintptr_t>(x) |
                        reinterpret_cast<uintptr_t>(rows);
  if (bits % 16 == 0) return RunToExperts<uint4>(x, stride, row, o, rows, s);
  if (bits % 8 == 0) return RunToExperts<uint2>(x, stride, row, o, rows, s);
  if (bits % 4 == 0) return RunToExperts<uint32_t>(x, stride, row, o, rows, s);
  return RunToExperts<uint16_t>(x, stride, row, o, rows, s);
}

int scemb_tokens_from_experts(const void* rows, int32_t type,
                              int64_t rows_stride, int64_t dim,
                              const void* weights, int32_t weights_type,
                              const scemb_expert_order_t* order, void* y,
                              void* stream) {
  using namespace scemb;
  const int bad = CheckOrder(order, type, dim);
  if (bad != 0) return bad;
  if (order->tokens == 0) return SCEMB_OK;
  if (rows == nullptr || y == nullptr || rows_stride < 0 ||
      (weights_type != SCEMB_F32 && weights_type != type)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "tokens from experts: rows or y missing, a negative stride, "
                "or weights that are neither float32 nor of rows' type");
  }
  const Order o = OrderOf(order);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = weights_type == SCEMB_F32;
  switch (type) {
    case SCEMB_F32:
      return FromExpertsOf<float>(rows, rows_stride, dim, weights, f32, o, y,
                                  s);
    case SCEMB_BF16:
      return FromExpertsOf<bf16>(rows, rows_stride, dim, weights, f32, o, y,
                                 s);
    default:
      return FromExpertsOf<f16>(rows, rows_stride, dim, weights, f32, o, y, s);
  }
}

int scemb_tokens_from_experts_grad(
    const void* y_grad, int64_t y_grad_stride, const void* rows, int32_t type,
    int64_t rows_stride, int64_t dim, const void* weights,
    int32_t weights_type, const scemb_expert_order_t* order, void* rows_grad,
    void* weights_grad, void* stream) {
  using namespace scemb;
  const int bad = CheckOrder(order, type, dim);
  if (bad != 0) return bad;
  if (order->tokens == 0) return SCEMB_OK;
  if (y_grad == nullptr || rows == nullptr || rows_grad == nullptr ||
      rows_stride < 0 || y_grad_stride < 0 ||
      (weights_type != SCEMB_F32 && weights_type != type)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "tokens from experts, gradient: an operand is missing, a "
                "negative stride, or weights that are neither float32 nor of "
                "rows' type");
  }
  const Order o = OrderOf(order);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = weights_type == SCEMB_F32;
  switch (type) {
    case SCEMB_F32:
      return FromExpertsGradOf<float>(y_grad, y_grad_stride, rows, rows_stride,
                                      dim, weights, f32, o, rows_grad,
                                      weights_grad, s);
    case SCEMB_BF16:
      return FromExpertsGradOf<bf16>(y_grad, y_grad_stride, rows, rows_stride,
                                     dim, weights, f32, o, rows_grad,
                                     weights_grad, s);
    default:
      return FromExpertsGradOf<f16>(y_grad, y_grad_stride, rows, rows_stride,
                                    dim, weights, f32, o, rows_grad,
                                    weights_grad, s);
  }
}

}  // extern "C"
