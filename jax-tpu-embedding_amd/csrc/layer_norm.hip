// Layer norm over the last dimension, its gradient and the reduction of the
// weight's and the bias's gradients over the rows.
//
// A row is read once into the registers of G neighbouring lanes (a part of a
// wavefront, a wavefront or a work-group), kept in its own type, and both
// statistics come from there: the mean first, then the mean square of what is
// left, which loses nothing where the mean is large against the deviation.
// The work is HBM-bound: 2 values moved per element forwards, 3 backwards.
#include <algorithm>

#include "dense.h"

namespace scemb {
namespace {

constexpr int kCus = 256;

template <typename T>
struct NormArgs {
  const T* x;
  T* y;
  const void* weight;
  const void* bias;
  float* mean;
  float* rstd;
  int64_t rows;
  int64_t stride;
  int32_t dim;
  bool weight_f32;
  float epsilon;
};

template <typename T>
struct NormGradArgs {
  const T* dy;
  const T* x;
  T* dx;
  const float* mean;
  const float* rstd;
  const void* weight;
  float* partial;  // [2][gridDim.x][dim]: weight, bias
  int64_t rows;
  int64_t dy_stride;
  int64_t stride;
  int32_t dim;
  bool weight_f32;
};

// V weights from `at` on as float32 (`p` NULL: `missing`).
template <typename T, int V>
__device__ __forceinline__ void LoadWeights(const void* p, bool f32, int at,
                                            float missing, float (&w)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = missing;
  } else if (f32 || sizeof(T) == 4) {
    constexpr int kPart = V < 4 ? V : 4;
#pragma unroll
    for (int j = 0; j < V; j += kPart) {
      const auto v = LoadVec<float, kPart>(static_cast<const float*>(p) + at +
                                           j);
#pragma unroll
      for (int k = 0; k < kPart; ++k) w[j + k] = v.v[k];
    }
  } else {
    const auto v = LoadVec<T, V>(static_cast<const T*>(p) + at);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = static_cast<float>(v.v[j]);
  }
}

// Sums of N values over the G lanes of a row. Above a wavefront the row has
// the whole work-group: `part` holds N * G / 64 floats, and two calls in a row
// need two of them.
template <int G, int N>
__device__ __forceinline__ void RowSum(float (&x)[N], float* part) {
  constexpr int kLanes = G < kWave ? G : kWave;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = LaneSum<kLanes>(x[i]);
  if constexpr (G > kWave) {
    constexpr int kWaves = G / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[i * kWaves + threadIdx.x / kWave] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += part[i * kWaves + w];
      x[i] = s;
    }
  }
}

constexpr int BlockOf(int g) { return g > 256 ? g : 256; }

template <typename T, int V, int NV, int G>
__global__ __launch_bounds__(BlockOf(G)) void NormForward(NormArgs<T> a) {
  constexpr int kRows = BlockOf(G) / G;
  constexpr int kParts = G > kWave ? G / kWave : 1;
  __shared__ float part[2 * kParts];
  const int lane = threadIdx.x % G;
  const float scale = 1.f / static_cast<float>(a.dim);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows +
                     threadIdx.x / G;
       row < a.rows; row += static_cast<int64_t>(gridDim.x) * kRows) {
    const T* src = a.x + row * a.stride;
    Vec<T, V> x[NV];
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) x[i] = LoadVec<T, V>(src + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + lane) * V < a.dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] += static_cast<float>(x[i].v[j]);
      }
    }
    RowSum<G>(sum, part);
    const float mean = sum[0] * scale;
    float sq[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + lane) * V < a.dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = static_cast<float>(x[i].v[j]) - mean;
          sq[0] = fmaf(d, d, sq[0]);
        }
      }
    }
    RowSum<G>(sq, part + kParts);
    const float rstd = rsqrtf(sq[0] * scale + a.epsilon);
    if (lane == 0) {
      if (a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    T* dst = a.y + row * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        float w[V], b[V];
        LoadWeights<T, V>(a.weight, a.weight_f32, c, 1.f, w);
        LoadWeights<T, V>(a.bias, a.weight_f32, c, 0.f, b);
        Vec<T, V> y;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xhat = (static_cast<float>(x[i].v[j]) - mean) * rstd;
          y.v[j] = static_cast<T>(fmaf(xhat, w[j], b[j]));
        }
        StoreVec<T, V>(dst + c, y);
      }
    }
  }
}

// Rows longer than the registers of a work-group: three passes, the last two
// mostly from L2.
template <typename T, int V>
__global__ __launch_bounds__(1024) void NormForwardLong(NormArgs<T> a) {
  constexpr int G = 1024;
  __shared__ float part[2 * (G / kWave)];
  const float scale = 1.f / static_cast<float>(a.dim);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* src = a.x + row * a.stride;
    float sum[1] = {0.f};
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.dim;
         c += G * V) {
      const auto x = LoadVec<T, V>(src + c);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += static_cast<float>(x.v[j]);
    }
    RowSum<G>(sum, part);
    const float mean = sum[0] * scale;
    float sq[1] = {0.f};
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.dim;
         c += G * V) {
      const auto x = LoadVec<T, V>(src + c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = static_cast<float>(x.v[j]) - mean;
        sq[0] = fmaf(d, d, sq[0]);
      }
    }
    RowSum<G>(sq, part + G / kWave);
    const float rstd = rsqrtf(sq[0] * scale + a.epsilon);
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[row] = mean;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    T* dst = a.y + row * a.dim;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.dim;
         c += G * V) {
      const auto x = LoadVec<T, V>(src + c);
      float w[V], b[V];
      LoadWeights<T, V>(a.weight, a.weight_f32, static_cast<int>(c), 1.f, w);
      LoadWeights<T, V>(a.bias, a.weight_f32, static_cast<int>(c), 0.f, b);
      Vec<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
        y.v[j] = static_cast<T>(fmaf(xhat, w[j], b[j]));
      }
      StoreVec<T, V>(dst + c, y);
    }
  }
}

// The G lanes of a row take every gridDim.x-th row and keep their columns'
// share of the weight's and the bias's gradients in registers; at the end
// the groups of a work-group are added in LDS, in their order, and the
// work-group's sums go to `partial`.
template <typename T, int V, int NV, int G>
__global__ __launch_bounds__(BlockOf(G)) void NormBackward(NormGradArgs<T> a) {
  constexpr int kBlock = BlockOf(G);
  constexpr int kGroups = kBlock / G;
  constexpr int kParts = G > kWave ? 2 * (G / kWave) : 1;
  __shared__ float part[2 * kParts];
  const int lane = threadIdx.x % G;
  const int group = threadIdx.x / G;
  const float scale = 1.f / static_cast<float>(a.dim);
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = dw[i][j] = db[i][j] = 0.f;
    if (c < a.dim) {
      LoadWeights<T, V>(a.weight, a.weight_f32, c, 1.f, w[i]);
    }
  }
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
       row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    Vec<T, V> x[NV], dy[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        x[i] = LoadVec<T, V>(a.x + row * a.stride + c);
        dy[i] = LoadVec<T, V>(a.dy + row * a.dy_stride + c);
      }
    }
    const float mean = a.mean[row];
    const float rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + lane) * V < a.dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float g = static_cast<float>(dy[i].v[j]);
          const float xhat = (static_cast<float>(x[i].v[j]) - mean) * rstd;
          const float h = g * w[i][j];
          sum[0] += h;
          sum[1] = fmaf(h, xhat, sum[1]);
          dw[i][j] = fmaf(g, xhat, dw[i][j]);
          db[i][j] += g;
        }
      }
    }
    RowSum<G>(sum, part + turn * kParts);
    turn ^= 1;
    const float along1 = sum[0] * scale;
    const float alongx = sum[1] * scale;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        Vec<T, V> dx;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xhat = (static_cast<float>(x[i].v[j]) - mean) * rstd;
          const float h = static_cast<float>(dy[i].v[j]) * w[i][j];
          dx.v[j] = static_cast<T>((h - along1 - xhat * alongx) * rstd);
        }
        StoreVec<T, V>(a.dx + row * a.dim + c, dx);
      }
    }
  }
  if (a.partial == nullptr) return;
  float* out[2] = {
      a.partial + static_cast<int64_t>(blockIdx.x) * a.dim,
      a.partial + (static_cast<int64_t>(gridDim.x) + blockIdx.x) * a.dim};
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          out[0][c + j] = dw[i][j];
          out[1][c + j] = db[i][j];
        }
      }
    }
  } else {
    constexpr int kCols = G * V * NV;
    __shared__ float all[kGroups * kCols];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          all[group * kCols + (i * G + lane) * V + j] =
              which == 0 ? dw[i][j] : db[i][j];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.dim; c += kBlock) {
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) s += all[g * kCols + c];
        out[which][c] = s;
      }
    }
  }
}

// Rows longer than the registers of a work-group: the gradient of x in two
// passes over the row.
template <typename T, int V>
__global__ __launch_bounds__(1024) void NormBackwardLong(NormGradArgs<T> a) {
  constexpr int G = 1024;
  constexpr int kParts = 2 * (G / kWave);
  __shared__ float part[2 * kParts];
  const float scale = 1.f / static_cast<float>(a.dim);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* px = a.x + row * a.stride;
    const T* pdy = a.dy + row * a.dy_stride;
    const float mean = a.mean[row];
    const float rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f};
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.dim;
         c += G * V) {
      const auto x = LoadVec<T, V>(px + c);
      const auto dy = LoadVec<T, V>(pdy + c);
      float w[V];
      LoadWeights<T, V>(a.weight, a.weight_f32, static_cast<int>(c), 1.f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
        const float h = static_cast<float>(dy.v[j]) * w[j];
        sum[0] += h;
        sum[1] = fmaf(h, xhat, sum[1]);
      }
    }
    RowSum<G>(sum, part + turn * kParts);
    turn ^= 1;
    const float along1 = sum[0] * scale;
    const float alongx = sum[1] * scale;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.dim;
         c += G * V) {
      const auto x = LoadVec<T, V>(px + c);
      const auto dy = LoadVec<T, V>(pdy + c);
      float w[V];
      LoadWeights<T, V>(a.weight, a.weight_f32, static_cast<int>(c), 1.f, w);
      Vec<T, V> dx;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
        const float h = static_cast<float>(dy.v[j]) * w[j];
        dx.v[j] = static_cast<T>((h - along1 - xhat * alongx) * rstd);
      }
      StoreVec<T, V>(a.dx + row * a.dim + c, dx);
    }
  }
}

// Their weight's and bias's gradients: a thread has V columns (blockIdx.x)
// and every gridDim.y-th row.
template <typename T, int V>
__global__ __launch_bounds__(256) void NormColumnsLong(NormGradArgs<T> a) {
  const int64_t c =
      (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (c >= a.dim) return;
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const auto x = LoadVec<T, V>(a.x + row * a.stride + c);
    const auto dy = LoadVec<T, V>(a.dy + row * a.dy_stride + c);
    const float mean = a.mean[row];
    const float rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float g = static_cast<float>(dy.v[j]);
      const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
      dw[j] = fmaf(g, xhat, dw[j]);
      db[j] += g;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.partial[static_cast<int64_t>(blockIdx.y) * a.dim + c + j] = dw[j];
    a.partial[(static_cast<int64_t>(gridDim.y) + blockIdx.y) * a.dim + c + j] =
        db[j];
  }
}

// Adds the work-groups' sums: 32 columns a work-group, the `parts` rows of
// sums in 8 slices that LDS joins in their order.
template <typename W>
__global__ __launch_bounds__(256) void NormReduce(const float* partial,
                                                  int32_t parts, int32_t dim,
                                                  W* dweight, W* dbias) {
  __shared__ float sums[8][32];
  W* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  const int col = threadIdx.x % 32;
  const int slice = threadIdx.x / 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + col;
  const float* src =
      partial + static_cast<int64_t>(blockIdx.y) * parts * dim + c;
  float s = 0.f;
  if (c < dim) {
#pragma unroll 4
    for (int p = slice; p < parts; p += 8) {
      s += src[static_cast<int64_t>(p) * dim];
    }
  }
  sums[slice][col] = s;
  __syncthreads();
  if (slice == 0 && c < dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][col];
    out[c] = static_cast<W>(s);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// How a row is laid out over lanes: G lanes of NV vectors each. The fewest
// lanes whose registers hold the row, G = 0 for a row that no work-group
// holds.
struct Layout {
  int g;
  int nv;
};

Layout ForwardLayout(int v, int64_t dim) {
  const int64_t n = CeilDiv(dim, v);
  if (v == 1) {
    return n <= 64      ? Layout{16, 4}
           : n <= 256   ? Layout{64, 4}
           : n <= 1024  ? Layout{64, 16}
           : n <= 4096  ? Layout{256, 16}
           : n <= 8192  ? Layout{1024, 8}
                        : Layout{0, 0};
  }
  return n <= 4      ? Layout{4, 1}
         : n <= 16   ? Layout{16, 1}
         : n <= 32   ? Layout{16, 2}
         : n <= 64   ? Layout{64, 1}
         : n <= 128  ? Layout{64, 2}
         : n <= 256  ? Layout{64, 4}
         : n <= 512  ? Layout{64, 8}
         : n <= 1024 ? Layout{256, 4}
         : n <= 2048 ? Layout{256, 8}
         : n <= 4096 ? Layout{1024, 4}
                     : Layout{0, 0};
}

// At most 16 values a lane: their weights and two sums stay in registers too.
Layout BackwardLayout(int v, int64_t dim) {
  const int64_t n = CeilDiv(dim, v);
  if (v == 1) {
    return n <= 64      ? Layout{16, 4}
           : n <= 256   ? Layout{64, 4}
           : n <= 1024  ? Layout{64, 16}
           : n <= 4096  ? Layout{256, 16}
           : n <= 8192  ? Layout{1024, 8}
                        : Layout{0, 0};
  }
  const int most = 16 / v;  // vectors a lane
  return n <= 4              ? Layout{4, 1}
         : n <= 16           ? Layout{16, 1}
         : n <= 32           ? Layout{16, 2}
         : n <= 64           ? Layout{64, 1}
         : n <= 128          ? Layout{64, 2}
         : n <= 64 * most    ? Layout{64, most}
         : n <= 512          ? Layout{256, 2}
         : n <= 256 * most   ? Layout{256, most}
         : n <= 2048         ? Layout{1024, 2}
                             : Layout{0, 0};
}

// Work-groups of the backward pass, and so rows of partial sums: four a CU
// (two of 1024 threads), each group of lanes at least one row, and no more
// bytes of sums written and read than a quarter of what the rows are.
int64_t BackwardParts(Layout l, int type_bytes, int64_t rows) {
  const int groups = l.g == 0 ? 1 : BlockOf(l.g) / l.g;
  const int64_t most = l.g == 1024 || l.g == 0 ? kCus : 4 * kCus;
  const int64_t by_rows = CeilDiv(rows, groups);
  const int64_t by_bytes =
      std::max<int64_t>(rows * type_bytes * 3 / (4 * 16), 32);
  return std::max<int64_t>(1, std::min({most, by_rows, by_bytes}));
}

template <typename T>
int VectorWidth(int64_t dim, int64_t stride_a, int64_t stride_b,
                std::initializer_list<const void*> data) {
  constexpr int V = 16 / sizeof(T);
  if (dim % V != 0 || stride_a % V != 0 || stride_b % V != 0) return 1;
  for (const void* p : data) {
    if (!AlignedTo(p, 16)) return 1;
  }
  return V;
}

template <typename T, int V, int NV, int G>
int LaunchForward(const NormArgs<T>& a, hipStream_t stream) {
  const int64_t blocks = CeilDiv(a.rows, BlockOf(G) / G);
  hipLaunchKernelGGL((NormForward<T, V, NV, G>),
                     dim3(static_cast<uint32_t>(
                         std::min<int64_t>(blocks, 0x7fffffff))),
                     dim3(BlockOf(G)), 0, stream, a);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T, int V, int NV, int G>
int LaunchBackward(const NormGradArgs<T>& a, int64_t parts,
                   hipStream_t stream) {
  hipLaunchKernelGGL((NormBackward<T, V, NV, G>),
                     dim3(static_cast<uint32_t>(parts)), dim3(BlockOf(G)), 0,
                     stream, a);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

#define SCEMB_LAYOUT(G_, NV_, CALL)    \
  if (l.g == G_ && l.nv == NV_) {      \
    constexpr int G = G_, NV = NV_;    \
    return CALL;                       \
  }

template <typename T>
int Forward(const NormArgs<T>& a, hipStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const int v = VectorWidth<T>(a.dim, a.stride, a.stride,
                               {a.x, a.y, a.weight, a.bias});
  const Layout l = ForwardLayout(v, a.dim);
  const dim3 grid(
      static_cast<uint32_t>(std::min<int64_t>(a.rows, 0x7fffffff)));
  if (v == 1) {
    constexpr int V = 1;
    SCEMB_LAYOUT(16, 4, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 4, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 16, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(256, 16, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(1024, 8, (LaunchForward<T, V, NV, G>(a, stream)))
    hipLaunchKernelGGL((NormForwardLong<T, V>), grid, dim3(1024), 0, stream,
                       a);
  } else {
    constexpr int V = kWide;
    SCEMB_LAYOUT(4, 1, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(16, 1, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(16, 2, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 1, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 2, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 4, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(64, 8, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(256, 4, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(256, 8, (LaunchForward<T, V, NV, G>(a, stream)))
    SCEMB_LAYOUT(1024, 4, (LaunchForward<T, V, NV, G>(a, stream)))
    hipLaunchKernelGGL((NormForwardLong<T, V>), grid, dim3(1024), 0, stream,
                       a);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T, int V>
int BackwardLong(const NormGradArgs<T>& a, int64_t parts, hipStream_t stream) {
  const dim3 grid(
      static_cast<uint32_t>(std::min<int64_t>(a.rows, 0x7fffffff)));
  hipLaunchKernelGGL((NormBackwardLong<T, V>), grid, dim3(1024), 0, stream, a);
  SCEMB_LAUNCH_CHECK();
  if (a.partial != nullptr) {
    hipLaunchKernelGGL(
        (NormColumnsLong<T, V>),
        dim3(static_cast<uint32_t>(CeilDiv(a.dim, 256 * V)),
             static_cast<uint32_t>(parts)),
        dim3(256), 0, stream, a);
    SCEMB_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T>
int BackwardRows(const NormGradArgs<T>& a, int v, Layout l, int64_t parts,
                 hipStream_t stream) {
  if (v == 1) {
    constexpr int V = 1;
    SCEMB_LAYOUT(16, 4, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    SCEMB_LAYOUT(64, 4, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    SCEMB_LAYOUT(64, 16, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    SCEMB_LAYOUT(256, 16, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    SCEMB_LAYOUT(1024, 8, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    return BackwardLong<T, V>(a, parts, stream);
  }
  constexpr int V = 16 / sizeof(T);
  SCEMB_LAYOUT(4, 1, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(16, 1, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(16, 2, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(64, 1, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(64, 2, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(256, 2, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  SCEMB_LAYOUT(1024, 2, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  if constexpr (V == 4) {
    SCEMB_LAYOUT(64, 4, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
    SCEMB_LAYOUT(256, 4, (LaunchBackward<T, V, NV, G>(a, parts, stream)))
  }
  return BackwardLong<T, V>(a, parts, stream);
}
#undef SCEMB_LAYOUT

int CheckNorm(int32_t type, int32_t weight_type, int64_t rows, int64_t dim) {
  if (TypeBytes(type) == 0 ||
      (weight_type != SCEMB_F32 && weight_type != type)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "layer norm: x is float32, bfloat16 or float16, weight and "
                "bias are float32 or x's type");
  }
  if (rows < 0 || dim < 1 || dim > 0x7fffffff - 65536) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "layer norm: rows below 0 or dim outside [1, 2^31 - 2^16)");
  }
  return 0;
}

template <typename T>
int RunForward(const void* x, int64_t rows, int64_t dim, int64_t stride,
               const void* weight, const void* bias, bool weight_f32,
               float epsilon, void* y, float* mean, float* rstd,
               hipStream_t stream) {
  NormArgs<T> a;
  a.x = static_cast<const T*>(x);
  a.y = static_cast<T*>(y);
  a.weight = weight;
  a.bias = bias;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.stride = stride;
  a.dim = static_cast<int32_t>(dim);
  a.weight_f32 = weight_f32;
  a.epsilon = epsilon;
  return Forward<T>(a, stream);
}

template <typename T, typename W>
int RunReduce(const float* partial, int64_t parts, int64_t dim, void* dweight,
              void* dbias, hipStream_t stream) {
  hipLaunchKernelGGL((NormReduce<W>),
                     dim3(static_cast<uint32_t>(CeilDiv(dim, 32)), 2),
                     dim3(256), 0, stream, partial,
                     static_cast<int32_t>(parts), static_cast<int32_t>(dim),
                     static_cast<W*>(dweight), static_cast<W*>(dbias));
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int RunBackward(const void* dy, int64_t dy_stride, const void* x,
                int64_t stride, int64_t rows, int64_t dim, const float* mean,
                const float* rstd, const void* weight, bool weight_f32,
                void* dx, void* dweight, void* dbias, void* workspace,
                size_t workspace_bytes, hipStream_t stream) {
  NormGradArgs<T> a;
  a.dy = static_cast<const T*>(dy);
  a.x = static_cast<const T*>(x);
  a.dx = static_cast<T*>(dx);
  a.mean = mean;
  a.rstd = rstd;
  a.weight = weight;
  a.rows = rows;
  a.dy_stride = dy_stride;
  a.stride = stride;
  a.dim = static_cast<int32_t>(dim);
  a.weight_f32 = weight_f32;
  const int v = VectorWidth<T>(dim, stride, dy_stride, {dy, x, dx, weight});
  const Layout l = BackwardLayout(v, dim);
  const int64_t parts = BackwardParts(l, sizeof(T), rows);
  Arena arena(workspace, workspace_bytes);
  a.partial = nullptr;
  if (dweight != nullptr || dbias != nullptr) {
    a.partial = arena.Take<float>(2 * parts * dim);
    if (workspace == nullptr || arena.overflow()) {
      return Fail(SCEMB_ERR_WORKSPACE,
                  "layer norm gradient: workspace missing or too small");
    }
  }
  if (rows > 0) {
    const int rc = BackwardRows<T>(a, v, l, parts, stream);
    if (rc != 0) return rc;
  }
  if (a.partial == nullptr) return 0;
  const int64_t sums = rows > 0 ? parts : 0;
  return weight_f32
             ? RunReduce<T, float>(a.partial, sums, dim, dweight, dbias,
                                   stream)
             : RunReduce<T, T>(a.partial, sums, dim, dweight, dbias, stream);
}

}  // namespace
}  // namespace scemb

extern "C" {

int scemb_layer_norm(const void* x, int32_t type, int64_t rows, int64_t dim,
                     int64_t x_stride, const void* weight, const void* bias,
                     int32_t weight_type, float epsilon, void* y, float* mean,
                     float* rstd, void* stream) {
  using namespace scemb;
  const int bad = CheckNorm(type, weight_type, rows, dim);
  if (bad != 0) return bad;
  if (rows == 0) return SCEMB_OK;
  if (x == nullptr || y == nullptr || x_stride < 0) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "layer norm: x or y missing, or a negative stride");
  }
  const bool f32 = weight_type == SCEMB_F32;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (type) {
    case SCEMB_F32:
      return RunForward<float>(x, rows, dim, x_stride, weight, bias, f32,
                               epsilon, y, mean, rstd, s);
    case SCEMB_BF16:
      return RunForward<bf16>(x, rows, dim, x_stride, weight, bias, f32,
                              epsilon, y, mean, rstd, s);
    default:
      return RunForward<f16>(x, rows, dim, x_stride, weight, bias, f32,
                             epsilon, y, mean, rstd, s);
  }
}

size_t scemb_layer_norm_grad_workspace_size(int32_t type, int64_t rows,
                                            int64_t dim) {
  using namespace scemb;
  if (CheckNorm(type, type, rows, dim) != 0) return 0;
  const int bytes = TypeBytes(type);
  // What a call needs depends on its alignment: the larger of the two.
  int64_t parts = 0;
  for (const int v : {1, 16 / bytes}) {
    parts = std::max(parts, BackwardParts(BackwardLayout(v, dim), bytes, rows));
  }
  Arena arena(nullptr, 0);
  arena.Take<float>(2 * parts * dim);
  return arena.used();
}

int scemb_layer_norm_grad(const void* y_grad, int64_t y_grad_stride,
                          const void* x, int64_t x_stride, int32_t type,
                          int64_t rows, int64_t dim, const float* mean,
                          const float* rstd, const void* weight,
                          int32_t weight_type, void* x_grad,
                          void* weight_grad, void* bias_grad, void* workspace,
                          size_t workspace_bytes, void* stream) {
  using namespace scemb;
  const int bad = CheckNorm(type, weight_type, rows, dim);
  if (bad != 0) return bad;
  if (rows > 0 && (y_grad == nullptr || x == nullptr || mean == nullptr ||
                   rstd == nullptr || x_grad == nullptr || x_stride < 0 ||
                   y_grad_stride < 0)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "layer norm gradient: an operand is missing, or a negative "
                "stride");
  }
  const bool f32 = weight_type == SCEMB_F32;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (type) {
    case SCEMB_F32:
      return RunBackward<float>(y_grad, y_grad_stride, x, x_stride, rows, dim,
                                mean, rstd, weight, f32, x_grad, weight_grad,
                                bias_grad, workspace, workspace_bytes, s);
    case SCEMB_BF16:
      return RunBackward<bf16>(y_grad, y_grad_stride, x, x_stride, rows, dim,
                               mean, rstd, weight, f32, x_grad, weight_grad,
                               bias_grad, workspace, workspace_bytes, s);
    default:
      return RunBackward<f16>(y_grad, y_grad_stride, x, x_stride, rows, dim,
                              mean, rstd, weight, f32, x_grad, weight_grad,
                              bias_grad, workspace, workspace_bytes, s);
  }
}

}  // extern "C"
