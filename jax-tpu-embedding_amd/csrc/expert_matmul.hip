// Rows in the order of their experts times each expert's weights, and the
// gradients of both.
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

// y[r] = x[r] * W[expert of r] for rows in segments; zeros for rows of none.
template <typename C>
__global__ __launch_bounds__(C::kThreads, 2) void RowsKernel(
    const typename C::T* x, int64_t x_stride, int32_t rows, int32_t depth,
    Weights w, int32_t columns, const int32_t* offsets, int32_t experts,
    typename C::T* y, TileGrid grid) {
  using T = typename C::T;
  __shared__ __attribute__((aligned(16))) char lds0[C::kLds];
  __shared__ __attribute__((aligned(16))) char lds1[C::kLds];
  int32_t tile, column;
  if (!grid.Tile(blockIdx.x, &tile, &column)) return;
  const RowTile t = FindRowTile<C::kM>(offsets, experts, rows, tile);
  if (t.segment < 0) return;
  column *= C::kN;
  const int m = min(t.end - t.row, C::kM);
  const int n = min(columns - column, C::kN);
  C c;
  const T* b = static_cast<const T*>(w.data) + t.segment * w.expert +
               (C::kAlongB == Along::kDepth ? column * w.stride : column);
  c.Run(x + t.row * x_stride, x_stride, m, b, w.stride, n,
        t.segment < experts ? depth : 0, lds0, lds1, NoScales{});
  c.Store(y + static_cast<int64_t>(t.row) * columns + column, columns, m, n,
          lds0);
}

// dw[e] = the sum over the segment's rows of x[r]^T dy[r], or part `split` of
// `splits` of the rows in float32.
template <typename C, typename Out>
__global__ __launch_bounds__(C::kThreads, 2) void WeightsKernel(
    const typename C::T* x, int64_t x_stride, int32_t inner,
    const typename C::T* dy, int64_t dy_stride, int32_t outer, int32_t rows,
    const int32_t* offsets, int32_t experts, Out* dw, int32_t splits,
    TileGrid grid) {
  __shared__ __attribute__((aligned(16))) char lds0[C::kLds];
  __shared__ __attribute__((aligned(16))) char lds1[C::kLds];
  int32_t tile, column;
  if (!grid.Tile(blockIdx.x, &tile, &column)) return;
  const int32_t tiles = (inner + C::kM - 1) / C::kM;
  const int32_t part = tile / tiles;
  const int32_t e = part / splits;
  const int32_t row = tile % tiles * C::kM;
  column *= C::kN;
  Segment s = SegmentOf(offsets, experts, rows, e);
  const int32_t steps = (s.end - s.begin + C::kDepth - 1) / C::kDepth;
  const int32_t each = (steps + splits - 1) / splits * C::kDepth;
  s.begin = min(s.begin + static_cast<int64_t>(part % splits) * each,
                static_cast<int64_t>(s.end));
  s.end = min(s.end, s.begin + each);
  const int m = min(inner - row, C::kM);
  const int n = min(outer - column, C::kN);
  C c;
  c.Run(x + s.begin * x_stride + row, x_stride, m,
        dy + s.begin * dy_stride + column, dy_stride, n, s.end - s.begin,
        lds0, lds1, NoScales{});
  c.Store(dw + (static_cast<int64_t>(part) * inner + row) * outer + column,
          outer, m, n, lds0);
}

// out[e][i] = the sum over the splits of part[e][split][i], in their order.
constexpr int kJoinBlock = 256;
template <typename T>
__global__ __launch_bounds__(kJoinBlock) void JoinParts(const float* parts,
                                                        int64_t size,
                                                        int32_t splits,
                                                        int32_t experts,
                                                        T* out) {
  constexpr int V = 4;
  const int64_t vectors = (size + V - 1) / V;
  for (int64_t v = static_cast<int64_t>(blockIdx.x) * kJoinBlock + threadIdx.x;
       v < vectors * experts;
       v += static_cast<int64_t>(gridDim.x) * kJoinBlock) {
    const int64_t e = v / vectors, i = v % vectors * V;
    const float* from = parts + e * splits * size + i;
    T* to = out + e * size + i;
    if (i + V <= size) {
      Vec<float, V> sum = LoadVec<float, V>(from);
      for (int s = 1; s < splits; ++s) {
        const auto x = LoadVec<float, V>(from + s * size);
#pragma unroll
        for (int j = 0; j < V; ++j) sum.v[j] += x.v[j];
      }
      Vec<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) y.v[j] = static_cast<T>(sum.v[j]);
      StoreVec<T, V>(to, y);
    } else {
      for (int j = 0; i + j < size; ++j) {
        float sum = from[j];
        for (int s = 1; s < splits; ++s) sum += from[s * size + j];
        to[j] = static_cast<T>(sum);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

constexpr int kCus = 256;

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
  hipStream_t stream;

  template <typename C>
  int Launch() const {
    const TileGrid grid(rows / C::kM + experts + 1, CeilDiv(columns, C::kN));
    if (grid.Groups() > MostGroups(C::kThreads)) return TooMany();
    hipLaunchKernelGGL(RowsKernel<C>, dim3(grid.Groups()), dim3(C::kThreads),
                       0, stream, x, x_stride, static_cast<int32_t>(rows),
                       static_cast<int32_t>(depth), w,
                       static_cast<int32_t>(columns), offsets, experts, y,
                       grid);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }

  // kB: which of the weights' dimensions is contiguous.
  template <Along kB>
  int Run() const {
    constexpr int kBytes = sizeof(T);
    const bool direct = Loadable(x, x_stride, kBytes) &&
                        Loadable(w.data, w.stride, kBytes) &&
                        w.expert * kBytes % 16 == 0 &&
                        depth * kBytes % 16 == 0 &&
                        (kB == Along::kDepth || columns * kBytes % 16 == 0);
    const bool small = rows <= 32ll * experts;
    if (!direct) {
      return small ? Launch<SmallTile<T, Along::kDepth, kB, false>>()
                   : Launch<MiddleTile<T, Along::kDepth, kB, false>>();
    }
    if (small) return Launch<SmallTile<T, Along::kDepth, kB, true>>();
    if constexpr (kBytes == 2) {
      if (rows >= 256ll * experts) {
        return Launch<LargeTile<T, Along::kDepth, kB>>();
      }
    }
    return Launch<MiddleTile<T, Along::kDepth, kB, true>>();
  }
};

// How the weights' gradient is cut: its tiles, and into how many parts each
// expert's rows, so that there is a work-group for every CU where the rows are
// enough.
struct WeightsPlan {
  bool large;
  int32_t splits;
};
WeightsPlan PlanWeights(int bytes, int64_t rows, int64_t inner, int64_t outer,
                        int32_t experts) {
  WeightsPlan p = {false, 1};
  const auto tiles = [&](int size) {
    return CeilDiv(inner, size) * CeilDiv(outer, size) * experts;
  };
  p.large = bytes == 2 && tiles(256) >= kCus;
  const int64_t have = tiles(p.large ? 256 : 128);
  const int64_t steps = rows / experts / (128 / bytes);
  const int64_t most = static_cast<int64_t>(
      (64 << 20) / (4.0 * experts * inner * outer));
  const int64_t splits =
      std::min({CeilDiv(2 * kCus, have), steps / 4, most, int64_t{1024}});
  p.splits = static_cast<int32_t>(std::max<int64_t>(splits, 1));
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
    const TileGrid grid(CeilDiv(inner, C::kM) * plan.splits * experts,
                        CeilDiv(outer, C::kN));
    if (grid.Groups() > MostGroups(C::kThreads)) return TooMany();
    hipLaunchKernelGGL((WeightsKernel<C, Out>), dim3(grid.Groups()),
                       dim3(C::kThreads), 0, stream, x, x_stride,
                       static_cast<int32_t>(inner), dy, dy_stride,
                       static_cast<int32_t>(outer), static_cast<int32_t>(rows),
                       offsets, experts, out, plan.splits, grid);
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
    if (plan.splits == 1) return Run<T>(dw);
    const int rc = Run<float>(parts);
    if (rc != 0) return rc;
    const int64_t size = inner * outer;
    const int64_t blocks = CeilDiv(CeilDiv(size, 4) * experts, kJoinBlock);
    hipLaunchKernelGGL(JoinParts<T>,
                       dim3(std::min(blocks, MostGroups(kJoinBlock))),
                       dim3(kJoinBlock), 0, stream, parts, size, plan.splits,
                       experts, dw);
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

int scemb_expert_matmul(const void* rows, int32_t type, int64_t rows_stride,
                        int64_t num_rows, int64_t inner, int64_t outer,
                        const void* weights, int64_t expert_stride,
                        int64_t inner_stride, int64_t outer_stride,
                        const int32_t* offsets, int32_t num_experts, void* y,
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
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    const bool along_outer = outer_stride == 1;
    const RowsCall<T> call = {
        static_cast<const T*>(rows), rows_stride, num_rows, inner,
        {weights, expert_stride, along_outer ? inner_stride : outer_stride},
        outer, offsets, num_experts, static_cast<T*>(y),
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
  if (plan.splits == 1) return 0;
  return static_cast<size_t>(plan.splits) * num_experts * inner * outer * 4;
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
