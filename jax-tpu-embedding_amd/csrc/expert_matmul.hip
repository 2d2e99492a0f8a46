// Rows in the order of their experts times each expert's weights, and the
// gradients of both: y[r] = x[r] W[e], dx[r] = dy[r] W[e]^T,
// dW[e] = sum of x[r]^T dy[r] over the expert's rows.
//
// A work-group makes a tile of one expert's result with matrix instructions
// (tiles.h). How many rows an expert has is known on the GPU alone: the launch
// has work-groups for the most tiles there can be (a partial one for every
// expert), each finds its own from the offsets, and those past the last end at
// once. The rows' gradient is the product with the weights' dimensions changed
// about, so only which dimension is contiguous makes different kernels.
//
// Many rows are bound by the matrix cores at the clock that the chip's power
// leaves them, few rows by the weights' bytes. Measured, bfloat16, 8192^3: 827 us
// weights by input (1.33 PFLOP/s; the library's dense product 806), 819 by output
// (716), the weights' gradient 818 (939). 64 experts with 0 to 32,378 of 131,072
// rows, 1024 x 4096: forwards 1.18 ms, of which about a quarter is writing 1.07
// GB between the products (the library's one dense product of these sizes 0.98);
// backwards 2.1 ms (0.75 and 1.11). 128 rows of 64 experts: 43 to 46 us, the
// weights of the experts that have any at HBM's rate. float32 8192^3: 7.6 ms, 0.92
// of the library's rate.
#include <algorithm>

#include "tiles.h"

namespace scemb {
namespace {

// ---------------------------------------------------------------------------
// The kernels.
// ---------------------------------------------------------------------------

struct Weights {
  const void* data;
  int64_t expert;  // stride of an expert
  int64_t stride;  // of the dimension that is not contiguous
};

// y[r] = x[r] * W[expert of r] for rows in segments; zeros for rows of none. With
// more than one split, the sums over that part of the depth, [splits, rows,
// columns].
template <typename C, typename Out>
__global__ __launch_bounds__(C::kThreads, 2) void RowsKernel(
    const typename C::T* x, int64_t x_stride, int32_t rows, int32_t depth,
    Weights w, int32_t columns, const int32_t* offsets, int32_t experts,
    Out* y, int32_t splits, TileGrid grid) {
  using T = typename C::T;
  __shared__ __attribute__((aligned(16))) char lds0[C::kLds];
  __shared__ __attribute__((aligned(16))) char lds1[C::kLds];
  int32_t tile, column;
  if (!grid.Tile(blockIdx.x, &tile, &column)) return;
  const RowTile t = FindRowTile(offsets, experts, rows, tile, C::kM);
  if (t.segment < 0) return;
  int32_t begin = 0, count = depth;
  if (splits > 1) {
    const int32_t across = grid.columns / splits;
    const int32_t split = column / across;
    column -= split * across;
    const int32_t steps = (depth + C::kDepth - 1) / C::kDepth;
    const int32_t each = (steps + splits - 1) / splits * C::kDepth;
    begin = min(split * each, depth);
    count = min(each, depth - begin);
    y += static_cast<int64_t>(split) * rows * columns;
  }
  column *= C::kN;
  const int m = min(t.end - t.row, C::kM);
  const int n = min(columns - column, C::kN);
  C c;
  const T* b = static_cast<const T*>(w.data) + t.segment * w.expert +
               (C::kAlongB == Along::kDepth ? column * w.stride + begin
                                            : column + begin * w.stride);
  c.Run(x + t.row * x_stride + begin, x_stride, m, depth, b, w.stride, n,
        C::kAlongB == Along::kDepth ? depth : columns,
        t.segment < experts ? count : 0, lds0, lds1, NoScales{});
  c.Store(y + static_cast<int64_t>(t.row) * columns + column, columns, m, n,
          lds0);
}

// y[i] = the sum over the splits of parts[split][i], in their order.
constexpr int kJoinBlock = 256;
template <typename T>
__global__ __launch_bounds__(kJoinBlock) void JoinSplits(const float* parts,
                                                         int64_t size,
                                                         int32_t splits, T* y) {
  constexpr int V = 4;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kJoinBlock +
                    threadIdx.x) * V;
       i < size; i += static_cast<int64_t>(gridDim.x) * kJoinBlock * V) {
    if (i + V <= size) {
      float sum[V] = {};
#pragma unroll 4
      for (int p = 0; p < splits; ++p) {
        const auto x = LoadVec<float, V>(parts + p * size + i);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += x.v[j];
      }
      Vec<T, V> v;
#pragma unroll
      for (int j = 0; j < V; ++j) v.v[j] = static_cast<T>(sum[j]);
      StoreVec<T, V>(y + i, v);
    } else {
      for (int64_t j = i; j < size; ++j) {
        float sum = 0.f;
        for (int p = 0; p < splits; ++p) sum += parts[p * size + j];
        y[j] = static_cast<T>(sum);
      }
    }
  }
}

// dw[e] = the sum over the segment's rows of x[r]^T dy[r]; with `piece` not 0
// that of each `piece` rows of a segment, one after another.
template <typename C, typename Out>
__global__ __launch_bounds__(C::kThreads, 2) void WeightsKernel(
    const typename C::T* x, int64_t x_stride, int32_t inner,
    const typename C::T* dy, int64_t dy_stride, int32_t outer, int32_t rows,
    const int32_t* offsets, int32_t experts, Out* dw, int32_t piece,
    bool ranked, TileGrid grid) {
  __shared__ __attribute__((aligned(16))) char lds0[C::kLds];
  __shared__ __attribute__((aligned(16))) char lds1[C::kLds];
  int32_t tile, column;
  if (!grid.Tile(blockIdx.x, &tile, &column)) return;
  const int32_t tiles = (inner + C::kM - 1) / C::kM;
  int32_t part = tile / tiles;
  const int32_t row = tile % tiles * C::kM;
  column *= C::kN;
  Segment s;
  if (piece != 0) {
    const RowTile t = FindRowTile(offsets, experts, rows, part, piece);
    if (t.segment < 0 || t.segment >= experts) return;
    s = {t.row, t.end - t.row > piece ? t.row + piece : t.end};
  } else {
    // The longest sums first: one that begins last is all that runs then (64
    // experts, the largest with a quarter of all rows: 1345 us in their order,
    // 1081 this way). Finding which costs a work-group a few microseconds: 64
    // experts of 2048 rows each, 1024 x 4096, take 1097 us and 1028 in their
    // order, and sums of fewer than 256 rows are not worth it (64 rows each, 512 x
    // 512: 20 us, in their order 12).
    if (ranked) part = ExpertOfRank(offsets, experts, rows, part);
    s = SegmentOf(offsets, experts, rows, part);
    s = {__builtin_amdgcn_readfirstlane(s.begin),
         __builtin_amdgcn_readfirstlane(s.end)};
  }
  const int m = min(inner - row, C::kM);
  const int n = min(outer - column, C::kN);
  C c;
  c.Run(x + s.begin * x_stride + row, x_stride, m, inner,
        dy + s.begin * dy_stride + column, dy_stride, n, outer,
        s.end - s.begin, lds0, lds1, NoScales{});
  c.Store(dw + (static_cast<int64_t>(part) * inner + row) * outer + column,
          outer, m, n, lds0);
}

// out[e] = the sum of the pieces of segment e, in their order; there are `most`
// of all, whatever the offsets hold.
template <typename T>
__global__ __launch_bounds__(kJoinBlock) void JoinPieces(
    const float* pieces, int64_t size, const int32_t* offsets, int32_t experts,
    int32_t rows, int32_t piece, int32_t most, T* out) {
  constexpr int V = 4;
  const int32_t e = blockIdx.y;
  const int64_t first =
      min(max(TilesBefore(offsets, experts, rows, e, piece), 0), most);
  const int32_t n = min(TilesOf(SegmentOf(offsets, experts, rows, e), piece),
                        most - static_cast<int32_t>(first));
  const float* from = pieces + first * size;
  T* to = out + e * size;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kJoinBlock +
                    threadIdx.x) * V;
       i < size; i += static_cast<int64_t>(gridDim.x) * kJoinBlock * V) {
    if (i + V <= size) {
      float sum[V] = {};
#pragma unroll 4
      for (int p = 0; p < n; ++p) {
        const auto x = LoadVec<float, V>(from + p * size + i);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += x.v[j];
      }
      Vec<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) y.v[j] = static_cast<T>(sum[j]);
      StoreVec<T, V>(to + i, y);
    } else {
      for (int64_t j = i; j < size; ++j) {
        float sum = 0.f;
        for (int p = 0; p < n; ++p) sum += from[p * size + j];
        to[j] = static_cast<T>(sum);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Whether rows of `stride` values can be loaded 16 bytes a lane at offsets of
// 32 bits within a panel of 256.
bool Loadable(const void* p, int64_t stride, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) |
          static_cast<uintptr_t>(stride) * bytes) % 16 == 0 &&
         stride * bytes < (1ll << 31) / 256;
}

int TooMany() {
  return Fail(SCEMB_ERR_INVALID_ARGUMENT,
              "expert matmul: more tiles than a launch takes");
}

// Into how many parts of the depth the product is cut: where small tiles, of
// which every expert that has rows has one at least, leave CUs without work and
// the sums are long enough to pay for a second launch (float32, 512 rows, 4096 x
// 128: 17 us, uncut 93; bfloat16, 1000 rows of 4 experts, 2048 x 256: 14 and 18).
int32_t SplitsOf(int bytes, int64_t rows, int64_t depth, int64_t columns,
                 int64_t experts) {
  const int64_t tiles = std::max(CeilDiv(rows, 32), std::min(rows, experts)) *
                        CeilDiv(columns, 128);
  const int64_t steps = CeilDiv(depth * bytes, 128);
  if (tiles == 0 || tiles >= kCus || steps < 16 ||
      !WorthSmall(rows, columns, experts)) {
    return 1;
  }
  return static_cast<int32_t>(std::max<int64_t>(
      std::min({CeilDiv(2 * kCus, tiles), steps / 4, int64_t{16}}), 1));
}

template <typename T>
struct RowsCall {
  const T* x;
  int64_t x_stride;
  int64_t rows;
  int64_t depth;
  Weights w;
  int64_t columns;
  const int32_t* offsets;
  int32_t experts;
  T* y;
  float* parts;
  int32_t splits;
  hipStream_t stream;

  template <typename C, typename Out>
  int Launch(Out* out) const {
    const TileGrid grid(rows / C::kM + experts + kNone,
                        CeilDiv(columns, C::kN) * splits);
    if (grid.Groups() > MostGroups(C::kThreads)) return TooMany();
    hipLaunchKernelGGL((RowsKernel<C, Out>), dim3(grid.Groups()),
                       dim3(C::kThreads), 0, stream, x, x_stride,
                       static_cast<int32_t>(rows), static_cast<int32_t>(depth),
                       w, static_cast<int32_t>(columns), offsets, experts, out,
                       splits, grid);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }

  template <typename C>
  int LaunchSmall() const {
    if (splits == 1) return Launch<C>(y);
    const int rc = Launch<C>(parts);
    if (rc != 0) return rc;
    const int64_t size = rows * columns;
    hipLaunchKernelGGL(
        JoinSplits<T>,
        dim3(static_cast<uint32_t>(std::min(CeilDiv(size, 4 * kJoinBlock),
                                            MostGroups(kJoinBlock)))),
        dim3(kJoinBlock), 0, stream, parts, size, splits, y);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }

  // kB: which of the weights' dimensions is contiguous.
  template <Along kB>
  int Run() const {
    constexpr int kBytes = sizeof(T);
    constexpr Along kDepth = Along::kDepth;
    const bool direct = Loadable(x, x_stride, kBytes) &&
                        Loadable(w.data, w.stride, kBytes) &&
                        w.expert * kBytes % 16 == 0 &&
                        depth * kBytes % 16 == 0 &&
                        (kB == kDepth || columns * kBytes % 16 == 0);
    if (WorthSmall(rows, columns, experts)) {
      return direct ? LaunchSmall<SmallTile<T, kDepth, kB, true>>()
                    : LaunchSmall<SmallTile<T, kDepth, kB, false>>();
    }
    if (!direct) return Launch<MiddleTile<T, kDepth, kB, false>>(y);
    if constexpr (kBytes == 2) {
      if (rows >= 256ll * experts && WorthLarge(rows, columns)) {
        return Launch<LargeTile<T, kDepth, kB>>(y);
      }
    }
    return Launch<MiddleTile<T, kDepth, kB, true>>(y);
  }
};

// How the weights' gradient is cut: its tiles, and into pieces of how many rows
// each expert's sum (0: none). Where tiles of 128 x 128 are fewer than two for
// every CU, so that there are four work-groups for each whatever the experts'
// shares. With more tiles no sum is cut, and a call takes as long as its longest
// one: 64 experts of 131,072 rows in all, 512 x 512, 96 us with 2048 rows each, 284
// where one has 12,659.
struct WeightsPlan {
  bool large;
  int32_t piece;
  int64_t pieces;  // at most
};
WeightsPlan PlanWeights(int bytes, int64_t rows, int64_t inner, int64_t outer,
                        int32_t experts) {
  WeightsPlan p = {false, 0, 0};
  const auto tiles = [&](int size) {
    return CeilDiv(inner, size) * CeilDiv(outer, size);
  };
  p.large = bytes == 2 && tiles(256) * experts >= kCus;
  if (p.large || tiles(128) * experts >= 2 * kCus) return p;
  // A piece is eight steps at least, and the pieces' sums 128 MB at most.
  const int64_t step = 128 / bytes;
  const int64_t room = (128ll << 20) / (4 * inner * outer) - experts;
  if (room < 1) return p;
  const int64_t piece =
      RoundUp(std::max({CeilDiv(rows * tiles(128), 4 * kCus), 8 * step,
                        CeilDiv(rows, room)}),
              step);
  if (rows <= piece) return p;
  p.piece = static_cast<int32_t>(piece);
  p.pieces = rows / piece + experts;
  return p;
}

template <typename T>
struct WeightsCall {
  const T* x;
  int64_t x_stride;
  const T* dy;
  int64_t dy_stride;
  int64_t rows;
  int64_t inner;
  int64_t outer;
  const int32_t* offsets;
  int32_t experts;
  T* dw;
  float* parts;
  WeightsPlan plan;
  hipStream_t stream;

  template <typename C, typename Out>
  int Launch(Out* out) const {
    // Every expert's tiles are spread over the XCDs, which take work-groups in
    // turn whatever they have to do.
    const int64_t down = CeilDiv(inner, C::kM), across = CeilDiv(outer, C::kN);
    const TileGrid grid(down * (plan.piece != 0 ? plan.pieces : experts),
                        across, std::min<int64_t>(down * across / 8, 32));
    if (grid.Groups() > MostGroups(C::kThreads)) return TooMany();
    hipLaunchKernelGGL((WeightsKernel<C, Out>), dim3(grid.Groups()),
                       dim3(C::kThreads), 0, stream, x, x_stride,
                       static_cast<int32_t>(inner), dy, dy_stride,
                       static_cast<int32_t>(outer), static_cast<int32_t>(rows),
                       offsets, experts, out, plan.piece,
                       experts <= kMostRanked && rows >= 256ll * experts, grid);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }

  template <typename Out>
  int Run(Out* out) const {
    constexpr int kBytes = sizeof(T);
    constexpr Along kOuter = Along::kOuter;
    const bool direct =
        Loadable(x, x_stride, kBytes) && Loadable(dy, dy_stride, kBytes) &&
        inner * kBytes % 16 == 0 && outer * kBytes % 16 == 0;
    if (!direct) return Launch<MiddleTile<T, kOuter, kOuter, false>>(out);
    if constexpr (kBytes == 2) {
      if (plan.large) return Launch<LargeTile<T, kOuter, kOuter>>(out);
    }
    return Launch<MiddleTile<T, kOuter, kOuter, true>>(out);
  }

  int Run() const {
    if (plan.piece == 0) return Run<T>(dw);
    const int rc = Run<float>(parts);
    if (rc != 0) return rc;
    const int64_t size = inner * outer;
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(
                        CeilDiv(size, 4 * kJoinBlock), 4096)),
                    static_cast<uint32_t>(experts));
    hipLaunchKernelGGL(JoinPieces<T>, grid, dim3(kJoinBlock), 0, stream, parts,
                       size, offsets, experts, static_cast<int32_t>(rows),
                       plan.piece, static_cast<int32_t>(plan.pieces), dw);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }
};

// Nonzero: an error, said.
int CheckSizes(int32_t type, int64_t rows, int64_t inner, int64_t outer,
               int32_t experts) {
  constexpr int64_t kMost = 0x7fffffff - 65536;
  if (TypeBytes(type) == 0 || rows < 0 || rows > kMost || inner < 1 ||
      inner > kMost || outer < 1 || outer > kMost || experts < 1 ||
      experts > SCEMB_MAX_EXPERTS) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "expert matmul: types other than float32, bfloat16 and "
                "float16, rows, inner or outer outside [1, 2^31 - 2^16) (rows "
                "may be 0), or experts outside [1, 1024]");
  }
  return 0;
}

}  // namespace
}  // namespace scemb

extern "C" {

size_t scemb_expert_matmul_workspace_size(int32_t type, int64_t num_rows,
                                          int64_t inner, int64_t outer,
                                          int32_t num_experts) {
  using namespace scemb;
  if (CheckSizes(type, num_rows, inner, outer, num_experts) != 0) return 0;
  const int32_t splits =
      SplitsOf(TypeBytes(type), num_rows, inner, outer, num_experts);
  return splits == 1 ? 0 : static_cast<size_t>(splits) * num_rows * outer * 4;
}

int scemb_expert_matmul(const void* rows, int32_t type, int64_t rows_stride,
                        int64_t num_rows, int64_t inner, int64_t outer,
                        const void* weights, int64_t expert_stride,
                        int64_t inner_stride, int64_t outer_stride,
                        const int32_t* offsets, int32_t num_experts, void* y,
                        void* workspace, size_t workspace_bytes,
                        void* stream) {
  using namespace scemb;
  const int bad = CheckSizes(type, num_rows, inner, outer, num_experts);
  if (bad != 0) return bad;
  if (num_rows == 0) return SCEMB_OK;
  if (rows == nullptr || weights == nullptr || offsets == nullptr ||
      y == nullptr || rows_stride < 0 || expert_stride < 0 ||
      inner_stride < 0 || outer_stride < 0 ||
      (inner_stride != 1 && outer_stride != 1)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "expert matmul: an operand is missing, a negative stride, or "
                "weights that are contiguous in neither inner nor outer");
  }
  const size_t need = scemb_expert_matmul_workspace_size(
      type, num_rows, inner, outer, num_experts);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return Fail(SCEMB_ERR_WORKSPACE, "expert matmul: workspace too small");
  }
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    const bool along_outer = outer_stride == 1;
    const RowsCall<T> call = {
        static_cast<const T*>(rows), rows_stride, num_rows, inner,
        {weights, expert_stride, along_outer ? inner_stride : outer_stride},
        outer, offsets, num_experts, static_cast<T*>(y),
        static_cast<float*>(workspace),
        SplitsOf(sizeof(T), num_rows, inner, outer, num_experts),
        static_cast<hipStream_t>(stream)};
    return along_outer ? call.template Run<Along::kOuter>()
                       : call.template Run<Along::kDepth>();
  };
  return type == SCEMB_F32    ? run(float{})
         : type == SCEMB_BF16 ? run(bf16{})
                              : run(f16{});
}

size_t scemb_expert_matmul_weights_grad_workspace_size(int32_t type,
                                                       int64_t num_rows,
                                                       int64_t inner,
                                                       int64_t outer,
                                                       int32_t num_experts) {
  using namespace scemb;
  if (CheckSizes(type, num_rows, inner, outer, num_experts) != 0) return 0;
  const WeightsPlan plan =
      PlanWeights(TypeBytes(type), num_rows, inner, outer, num_experts);
  return static_cast<size_t>(plan.pieces) * inner * outer * 4;
}

int scemb_expert_matmul_weights_grad(
    const void* rows, int64_t rows_stride, const void* y_grad,
    int64_t y_grad_stride, int32_t type, int64_t num_rows, int64_t inner,
    int64_t outer, const int32_t* offsets, int32_t num_experts,
    void* weights_grad, void* workspace, size_t workspace_bytes,
    void* stream) {
  using namespace scemb;
  const int bad = CheckSizes(type, num_rows, inner, outer, num_experts);
  if (bad != 0) return bad;
  if ((num_rows > 0 && (rows == nullptr || y_grad == nullptr)) ||
      offsets == nullptr || weights_grad == nullptr || rows_stride < 0 ||
      y_grad_stride < 0) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "expert matmul, weights' gradient: an operand is missing, or a "
                "negative stride");
  }
  const size_t need = scemb_expert_matmul_weights_grad_workspace_size(
      type, num_rows, inner, outer, num_experts);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return Fail(SCEMB_ERR_WORKSPACE,
                "expert matmul, weights' gradient: workspace too small");
  }
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    const WeightsCall<T> call = {
        static_cast<const T*>(rows), rows_stride,
        static_cast<const T*>(y_grad), y_grad_stride, num_rows, inner, outer,
        offsets, num_experts, static_cast<T*>(weights_grad),
        static_cast<float*>(workspace),
        PlanWeights(sizeof(T), num_rows, inner, outer, num_experts),
        static_cast<hipStream_t>(stream)};
    return call.Run();
  };
  return type == SCEMB_F32    ? run(float{})
         : type == SCEMB_BF16 ? run(bf16{})
                              : run(f16{});
}

}  // extern "C"
