// Tokens ordered by expert and back: a stable counting sort of the choices,
// the copy of the tokens' rows to their places, the weighted sum of the rows
// back at their tokens, and the gradients.
//
// The sort knows both where a choice goes (positions) and where it came from
// (sources), so every kernel works token by token: it reads a token's row once
// however many choices it has (the weighted sum's gradient loads it for each
// choice, the first time from memory, then from the caches), writes whole rows,
// and sums in the order of the choices. Nothing is added atomically. (Row by row
// of the experts' order, a token's row would be read once for each choice, from
// anywhere.)
//
// The sort is latency: 131,072 choices are 3 MB, and take 5 us to count and 7
// to place. The rows are HBM-bound. Measured, 65,536 tokens with two of 64
// experts each and 1024 bfloat16 columns: to the experts 76 us (5.3 TB/s) after
// 11 us of sorting, back 67 us (6.0 TB/s); the gradient of four choices of
// 16,384 tokens with 512 columns 30 us (5.1 TB/s).
#include <algorithm>

#include "dense.h"

namespace scemb {
namespace {

// ---------------------------------------------------------------------------
// Counting sort.
// ---------------------------------------------------------------------------

constexpr int kTileWaves = 4;        // work-group of a tile
constexpr int kSingleWaves = 16;     // work-group of a sort in one launch
// Ids of a tile, or a multiple of it (131,072 ids: three launches of 19 us in
// tiles of 2048, 15 in these).
constexpr int64_t kTile = 1024;
constexpr int64_t kMaxTiles = 4096;  // counts of all tiles are scanned
// Up to here one work-group sorts by itself in one launch, where its counts fit
// 64 KB of LDS (6000 ids 9.1 us against 10.9 in two launches, 8000 10.9 and
// 11.0, 12,000 14.7 and 10.9).
constexpr int64_t kSingle = 8192;
// Counts of all tiles up to which every tile adds them up itself, in two
// launches instead of three (131,072 ids of 64 experts, 8192 counts: 11.0 us
// against 13.9; 60,000 of 256, 15,104 counts: 12.9 and 14.2; 300,000 of 64,
// 18,752 counts: 14.6 and 13.9).
constexpr int64_t kOwnSumsMost = 16384;
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

// The keys of choices i, i + step, ... (kNoKey from `last` > 0 on), kKeys loads
// in flight: one by one, each waits for memory.
constexpr int kKeys = 4;
constexpr uint32_t kNoKey = ~0u;
template <typename I>
__device__ __forceinline__ void LoadKeys(const I* ids, int32_t experts,
                                         int64_t i, int64_t step, int64_t last,
                                         uint32_t (&keys)[kKeys]) {
#pragma unroll
  for (int k = 0; k < kKeys; ++k) {
    const int64_t at = i + k * step;
    keys[k] = KeyOf(ids, at < last ? at : last - 1, experts);
  }
#pragma unroll
  for (int k = 0; k < kKeys; ++k) {
    if (i + k * step >= last) keys[k] = kNoKey;
  }
}

// Adds the keys of choices i, i + step, ... to `counts` in LDS.
template <typename I>
__device__ __forceinline__ void CountKeys(const I* ids, int32_t experts,
                                          int64_t i, int64_t step,
                                          int64_t last, uint32_t* counts) {
  for (; i < last; i += kKeys * step) {
    uint32_t keys[kKeys];
    LoadKeys(ids, experts, i, step, last, keys);
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      if (keys[k] != kNoKey) atomicAdd(&counts[keys[k]], 1u);
    }
  }
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
  CountKeys(ids, experts, first + threadIdx.x % kWave, kWave, last,
            counts + (threadIdx.x / kWave) * row);
  __syncthreads();
}

// Places a wavefront's share: next[key] is the place of its next choice of
// that key. 64 choices at a time, equal keys ranked by lane.
template <typename I>
__device__ __forceinline__ void PlaceShare(const I* ids, int64_t n,
                                           int32_t experts, int64_t first,
                                           int64_t last, uint32_t* next,
                                           int32_t* positions,
                                           int32_t* sources) {
  const int lane = threadIdx.x % kWave;
  for (int64_t at = first; at < last; at += kKeys * kWave) {
    uint32_t keys[kKeys];
    LoadKeys(ids, experts, at + lane, kWave, last, keys);
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      if (at + k * kWave >= last) break;  // uniform
      const uint32_t key = keys[k];
      const bool in = key != kNoKey;
      const uint64_t same = MatchLanes<kKeyBits>(__ballot(in), key);
      const int leader =
          in ? __ffsll(static_cast<unsigned long long>(same)) - 1 : lane;
      uint32_t base = 0;
      if (in && lane == leader) {
        base = atomicAdd(&next[key], static_cast<uint32_t>(__popcll(same)));
      }
      base = __shfl(base, leader, kWave);
      if (in) {
        const int64_t i = at + k * kWave + lane;
        const uint32_t place = base + __popcll(same & LaneMaskLt());
        positions[i] = static_cast<int32_t>(place);
        // Always, unless the ids changed since they were counted.
        if (place < n) sources[place] = static_cast<int32_t>(i);
      }
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
  PlaceShare(ids, n, experts, s.first, s.last,
             counts + (threadIdx.x / kWave) * row, positions, sources);
}

// Counts of each tile: hist[tile][key] where the tiles add them up themselves
// (kOwnSums), hist[key][tile] for ScanTiles.
template <typename I, bool kOwnSums>
__global__ __launch_bounds__(kTileWaves* kWave) void CountTiles(
    const I* ids, int64_t n, int32_t experts, int64_t tile, uint32_t* hist) {
  constexpr int kBlock = kTileWaves * kWave;
  extern __shared__ uint32_t counts[];
  const int row = experts + 1;
  for (int i = threadIdx.x; i < row; i += kBlock) counts[i] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * tile;
  const int64_t end = begin + tile < n ? begin + tile : n;
  CountKeys(ids, experts, begin + threadIdx.x, kBlock, end, counts);
  __syncthreads();
  for (int i = threadIdx.x; i < row; i += kBlock) {
    const int64_t at = kOwnSums ? static_cast<int64_t>(blockIdx.x) * row + i
                                : static_cast<int64_t>(i) * gridDim.x +
                                      blockIdx.x;
    hist[at] = counts[i];
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

// Turns the counts of a tile's wavefronts for key e into the places of their
// first choices; `place` is the tile's.
__device__ __forceinline__ void PlacesOf(uint32_t* counts, int row, int e,
                                         uint32_t place) {
#pragma unroll
  for (int w = 0; w < kTileWaves; ++w) {
    const uint32_t c = counts[w * row + e];
    counts[w * row + e] = place;
    place += c;
  }
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
    uint32_t sum = 0;
    const uint32_t before =
        run + BlockExclusiveScan<uint32_t, kBlock>(e < row ? totals[e] : 0u,
                                                   scan, &sum);
    run += sum;
    if (e < row) {
      if (blockIdx.x == 0) offsets[e] = static_cast<int32_t>(before);
      PlacesOf(counts, row, e,
               before +
                   hist[static_cast<int64_t>(e) * gridDim.x + blockIdx.x]);
    }
  }
  __syncthreads();
  PlaceShare(ids, n, experts, s.first, s.last,
             counts + (threadIdx.x / kWave) * row, positions, sources);
}

// The same without ScanTiles: every work-group adds up the counts of all tiles
// itself, 2^lanes_log threads (at least the experts) a slice of the tiles. The
// dropped choices before a tile are those that are left.
template <typename I>
__global__ __launch_bounds__(kTileWaves* kWave) void SumAndPlaceTiles(
    const I* ids, int64_t n, int32_t experts, int32_t lanes_log, int64_t tile,
    const uint32_t* hist, int32_t* positions, int32_t* sources,
    int32_t* offsets) {
  constexpr int kBlock = kTileWaves * kWave;
  extern __shared__ uint32_t counts[];
  __shared__ uint32_t scan[kTileWaves + 1];
  __shared__ uint32_t before_of[kBlock], total_of[kBlock];
  const int row = experts + 1;
  const int64_t begin = blockIdx.x * tile;
  const int64_t end = begin + tile < n ? begin + tile : n;
  const Share s = ShareOf<kTileWaves>(begin, end);
  const int e = threadIdx.x & ((1 << lanes_log) - 1);
  const uint32_t slices = kBlock >> lanes_log;
  uint32_t before = 0, total = 0;
  if (e < experts) {
    constexpr int kLoads = 8;  // in flight
    for (uint32_t t = threadIdx.x >> lanes_log; t < gridDim.x;
         t += kLoads * slices) {
      uint32_t c[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t u = t + i * slices;
        c[i] = u < gridDim.x ? hist[u * row + e] : 0u;
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        total += c[i];
        before += t + i * slices < blockIdx.x ? c[i] : 0u;
      }
    }
  }
  before_of[threadIdx.x] = before;
  total_of[threadIdx.x] = total;
  CountShares<I, kTileWaves>(ids, experts, s.first, s.last, counts);
  before = total = 0;
  if (threadIdx.x < experts) {
    for (int i = threadIdx.x; i < kBlock; i += 1 << lanes_log) {
      before += before_of[i];
      total += total_of[i];
    }
  }
  uint32_t kept = 0, kept_before = 0;
  const uint32_t first =
      BlockExclusiveScan<uint32_t, kBlock>(total, scan, &kept);
  BlockExclusiveScan<uint32_t, kBlock>(before, scan, &kept_before);
  if (threadIdx.x < experts) {
    if (blockIdx.x == 0) offsets[threadIdx.x] = static_cast<int32_t>(first);
    PlacesOf(counts, row, threadIdx.x, first + before);
  }
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) offsets[experts] = static_cast<int32_t>(kept);
    PlacesOf(counts, row, experts,
             kept + static_cast<uint32_t>(begin) - kept_before);
  }
  __syncthreads();
  PlaceShare(ids, n, experts, s.first, s.last,
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
  const dim3 block(kTileWaves * kWave);
  const int lanes_log = BitWidth(experts - 1);
  if ((1 << lanes_log) <= kTileWaves * kWave &&
      (static_cast<int64_t>(tiles) << lanes_log) <= kOwnSumsMost) {
    hipLaunchKernelGGL((CountTiles<I, true>), dim3(tiles), block, row, stream,
                       in, n, experts, tile, hist);
    SCEMB_LAUNCH_CHECK();
    hipLaunchKernelGGL(SumAndPlaceTiles<I>, dim3(tiles), block,
                       kTileWaves * row, stream, in, n, experts, lanes_log, tile,
                       hist, positions, sources, offsets);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }
  hipLaunchKernelGGL((CountTiles<I, false>), dim3(tiles), block, row, stream,
                     in, n, experts, tile, hist);
  SCEMB_LAUNCH_CHECK();
  hipLaunchKernelGGL(ScanTiles, dim3((experts + 4) / 4), dim3(256), 0, stream,
                     hist, static_cast<int32_t>(tiles), experts + 1, totals);
  SCEMB_LAUNCH_CHECK();
  hipLaunchKernelGGL(PlaceTiles<I>, dim3(tiles), block, kTileWaves * row,
                     stream, in, n, experts, tile, hist,
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

  // Choices that are kept, within what there are whatever the order says.
  __device__ __forceinline__ uint32_t Kept() const {
    const int64_t n = tokens * choices;
    const int64_t k = *kept;
    return static_cast<uint32_t>(k < 0 ? 0 : k < n ? k : n);
  }
};

// E: an unsigned type of the elements' size; they are only moved.
template <typename E, int G, Cut kCut, bool kStream>
__global__ __launch_bounds__(kRowBlock) void ToExperts(const E* x,
                                                       int64_t stride,
                                                       int32_t dim,
                                                       Order order, E* rows) {
  constexpr int V = kVec<E>;
  constexpr int kTokens = kRowBlock / G;
  const int lane = threadIdx.x % G;
  const uint32_t kept = order.Kept();
  const uint32_t all = static_cast<uint32_t>(order.tokens * order.choices);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens +
                   threadIdx.x / G;
       t < order.tokens; t += static_cast<int64_t>(gridDim.x) * kTokens) {
    const int32_t* places = order.positions + t * order.choices;
    for (int32_t c = lane * V; c < dim; c += G * V) {
      const Span<kCut, V> s(c, dim);
      const auto v = LoadSpan<kCut, E, V, kStream>(x + t * stride, s);
      for (int k = 0; k < order.choices; ++k) {
        const uint32_t p = static_cast<uint32_t>(places[k]);
        if (p < all) {  // always, in an order that a sort made
          StoreSpan<kCut, E, V>(rows + static_cast<int64_t>(p) * dim, s,
                                p < kept ? v : Vec<E, V>{});
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

template <typename T, int G, Cut kCut, bool kStream>
__global__ __launch_bounds__(kRowBlock) void FromExperts(
    const T* rows, int64_t stride, int32_t dim, const void* weights,
    bool weights_f32, Order order, T* y) {
  constexpr int V = kVec<T>;
  constexpr int kTokens = kRowBlock / G;
  const int lane = threadIdx.x % G;
  const uint32_t kept = order.Kept();
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens +
                   threadIdx.x / G;
       t < order.tokens; t += static_cast<int64_t>(gridDim.x) * kTokens) {
    const int64_t first = t * order.choices;
    for (int32_t c = lane * V; c < dim; c += G * V) {
      const Span<kCut, V> s(c, dim);
      float sum[V];
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.f;
#pragma unroll 2
      for (int k = 0; k < order.choices; ++k) {
        const uint32_t p = static_cast<uint32_t>(order.positions[first + k]);
        if (p < kept) {
          const float w = WeightAt<T>(weights, weights_f32, first + k);
          const auto v =
              LoadSpan<kCut, T, V, kStream>(rows + p * stride, s);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            sum[j] = fmaf(w, static_cast<float>(v.v[j]), sum[j]);
          }
        }
      }
      Vec<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) out.v[j] = static_cast<T>(sum[j]);
      StoreSpan<kCut, T, V>(y + t * dim, s, out);
    }
  }
}

template <typename T, int G, Cut kCut>
__global__ __launch_bounds__(kRowBlock) void FromExpertsGrad(
    const T* dy, int64_t dy_stride, const T* rows, int64_t stride, int32_t dim,
    const void* weights, bool weights_f32, Order order, T* drows,
    void* dweights) {
  constexpr int V = kVec<T>;
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
          const Span<kCut, V> s(c, dim);
          Vec<T, V> out;
          if (keep) {
            const auto g = LoadSpan<kCut, T, V>(dy + t * dy_stride, s);
            const auto v = LoadSpan<kCut, T, V>(rows + p * stride, s);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float gj = static_cast<float>(g.v[j]);
              const float r =
                  s.Has(j) ? static_cast<float>(v.v[j]) : 0.f;
              dot = fmaf(s.Has(j) ? gj : 0.f, r, dot);
              out.v[j] = static_cast<T>(w * gj);
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = static_cast<T>(0.f);
          }
          StoreSpan<kCut, T, V>(drows + static_cast<int64_t>(p) * dim, s, out);
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
      std::min(CeilDiv(tokens, kRowBlock / g), MostGroups(kRowBlock)));
}

// Launches `kernel` with the fewest lanes a token, from 8 to a wavefront, that
// hold its row at a vector each: lanes past a row's end do nothing (100 float32
// columns of 20,011 tokens' three choices: 10.9 us with 64 lanes, 9.2 with 32).
#define SCEMB_LANES_OF(G_, CUT_, kernel, ...)                               \
  {                                                                         \
    constexpr int G = G_;                                                   \
    constexpr Cut kCut = CUT_;                                              \
    hipLaunchKernelGGL(kernel, dim3(RowGrid(o.tokens, G)), dim3(kRowBlock), \
                       0, stream, __VA_ARGS__);                             \
  }
#define SCEMB_LANES_CUT(CUT_, v, kernel, ...)      \
  if (dim <= 8 * (v)) {                            \
    SCEMB_LANES_OF(8, CUT_, kernel, __VA_ARGS__)   \
  } else if (dim <= 16 * (v)) {                    \
    SCEMB_LANES_OF(16, CUT_, kernel, __VA_ARGS__)  \
  } else if (dim <= 32 * (v)) {                    \
    SCEMB_LANES_OF(32, CUT_, kernel, __VA_ARGS__)  \
  } else {                                         \
    SCEMB_LANES_OF(64, CUT_, kernel, __VA_ARGS__)  \
  }
#define SCEMB_LANES(v, kernel, ...)                                \
  if (CutOf(dim, v) == Cut::kPart) {                               \
    SCEMB_LANES_OF(8, Cut::kPart, kernel, __VA_ARGS__)             \
  } else if (CutOf(dim, v) == Cut::kOver) {                        \
    SCEMB_LANES_CUT(Cut::kOver, v, kernel, __VA_ARGS__)            \
  } else {                                                         \
    SCEMB_LANES_CUT(Cut::kWhole, v, kernel, __VA_ARGS__)           \
  }                                                                \
  SCEMB_LAUNCH_CHECK();

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

// Whether the tokens' and the choices' rows are more than the last cache.
bool PastCache(const Order& o, int64_t dim, int64_t bytes) {
  return o.tokens * (o.choices + 1) * dim * bytes > kCacheBytes;
}

template <typename E>
int RunToExperts(const void* x, int64_t stride, int64_t dim, const Order& o,
                 void* rows, hipStream_t stream) {
  const E* from = static_cast<const E*>(x);
  E* to = static_cast<E*>(rows);
  const int32_t d = static_cast<int32_t>(dim);
  if (PastCache(o, dim, sizeof(E))) {
    SCEMB_LANES(kVec<E>, (ToExperts<E, G, kCut, true>), from, stride, d, o, to)
  } else {
    SCEMB_LANES(kVec<E>, (ToExperts<E, G, kCut, false>), from, stride, d, o,
                to)
  }
  return 0;
}

template <typename T>
int RunFromExperts(const void* rows, int64_t stride, int64_t dim,
                   const void* weights, bool f32, const Order& o, void* y,
                   hipStream_t stream) {
  const T* from = static_cast<const T*>(rows);
  T* to = static_cast<T*>(y);
  const int32_t d = static_cast<int32_t>(dim);
  if (PastCache(o, dim, sizeof(T))) {
    SCEMB_LANES(kVec<T>, (FromExperts<T, G, kCut, true>), from, stride, d,
                weights, f32, o, to)
  } else {
    SCEMB_LANES(kVec<T>, (FromExperts<T, G, kCut, false>), from, stride, d,
                weights, f32, o, to)
  }
  return 0;
}

template <typename T>
int RunFromExpertsGrad(const void* dy, int64_t dy_stride, const void* rows,
                       int64_t stride, int64_t dim, const void* weights,
                       bool f32, const Order& o, void* drows, void* dweights,
                       hipStream_t stream) {
  SCEMB_LANES(kVec<T>, (FromExpertsGrad<T, G, kCut>),
              static_cast<const T*>(dy), dy_stride,
              static_cast<const T*>(rows), stride, static_cast<int32_t>(dim),
              weights, f32, o, static_cast<T*>(drows), dweights)
  return 0;
}

}  // namespace
}  // namespace scemb

extern "C" {

size_t scemb_sort_by_expert_workspace_size(int64_t n, int32_t num_experts) {
  using namespace scemb;
  if (n < 0 || n > 0x7fffffff || num_experts < 1 ||
      num_experts > SCEMB_MAX_EXPERTS) {
    return 0;
  }
  Arena arena(nullptr, 0);
  if (!SortsSingle(n, num_experts)) {
    arena.Take<uint32_t>((num_experts + 1) * TilesOf(n));
    arena.Take<uint32_t>(num_experts + 1);
  }
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
  return TypeBytes(type) == 4
             ? RunToExperts<uint32_t>(x, x_stride, dim, o, rows, s)
             : RunToExperts<uint16_t>(x, x_stride, dim, o, rows, s);
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
      return RunFromExperts<float>(rows, rows_stride, dim, weights, f32, o, y,
                                  s);
    case SCEMB_BF16:
      return RunFromExperts<bf16>(rows, rows_stride, dim, weights, f32, o, y,
                                 s);
    default:
      return RunFromExperts<f16>(rows, rows_stride, dim, weights, f32, o, y, s);
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
      return RunFromExpertsGrad<float>(y_grad, y_grad_stride, rows, rows_stride,
                                      dim, weights, f32, o, rows_grad,
                                      weights_grad, s);
    case SCEMB_BF16:
      return RunFromExpertsGrad<bf16>(y_grad, y_grad_stride, rows, rows_stride,
                                     dim, weights, f32, o, rows_grad,
                                     weights_grad, s);
    default:
      return RunFromExpertsGrad<f16>(y_grad, y_grad_stride, rows, rows_stride,
                                    dim, weights, f32, o, rows_grad,
                                    weights_grad, s);
  }
}

}  // extern "C"
