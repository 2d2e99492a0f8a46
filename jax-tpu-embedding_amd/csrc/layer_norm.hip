// Layer norm over the last dimension, its gradient and the reduction of the
// weight's and the bias's gradients over the rows.
//
// A row is read once into the registers of G neighbouring lanes (a part of a
// wavefront, a wavefront or a work-group), kept in its own type, and both
// statistics come from there: a first mean, then the sums of what is left and
// of its squares. What is left has a mean of its own, the first one's rounding:
// with d = x - first, shift = mean(d),
//   mean = first + shift, variance = mean(d^2) - shift^2,
//   xhat = d * rstd - shift * rstd,
// or every xhat of a row whose mean is large against its deviations would be
// off by shift * rstd (1024 values of 10,000.3: 0.7 instead of 0). The mean
// that is returned is float32, and the gradient takes it as it is.
// Backwards, h = w * dy loses its mean and its part along xhat,
//   dx = rstd * (h - mean(h) - xhat * mean(h * xhat)),
// which takes one pass over the row's registers for both means and one for dx.
//
// Both are HBM-bound: 2 values moved per element forwards, 3 backwards, and
// what the lanes compute fits beside it (VALU busy 0.65 forwards). Measured,
// bfloat16 rows with float32 weights: 65,536 x 3328 forwards 165 us, 5.3 TB/s;
// 65,536 x 1024 backwards 75 us with the reduction, 5.4 TB/s; a device copy
// moves 4.9 TB/s.
#include <algorithm>

#include "dense.h"

namespace scemb {
namespace {

constexpr int kCus = 256;
// Threads of a CU forwards, about twice what it holds: from 1024 to 8192 times
// differ by 2 to 8%, wide rows gaining from more and 262,144 x 64 losing 20%
// below 1536.
constexpr int kForwardThreads = 4096;

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

// A vector's weights as float32 (`p` NULL: `missing`).
template <Cut kCut, typename T, int V>
__device__ __forceinline__ void LoadWeights(const void* p, bool f32,
                                            const Span<kCut, V>& s,
                                            float missing, float (&w)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = missing;
  } else if (f32 || sizeof(T) == 4) {
    const float* q = static_cast<const float*>(p);
    if constexpr (kCut == Cut::kPart) {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = j < s.hi ? q[j] : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const auto v = LoadVec<float, 4>(q + s.at + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[j + k] = v.v[k];
      }
    }
  } else {
    const auto v = LoadSpan<kCut, T, V>(static_cast<const T*>(p), s);
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
      if constexpr (kWaves > 4) {
        // A lane reads one wavefront's sum and the lanes join them, in four
        // steps instead of 16 (16,384 x 8192 bfloat16 forwards 106 us by
        // steps of one and 101, backwards 180 and 174; but with four sums
        // 32,768 x 2048 backwards 89 and 91).
        x[i] = LaneSum<kWaves>(part[i * kWaves + threadIdx.x % kWaves]);
      } else {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s += part[i * kWaves + w];
        x[i] = s;
      }
    }
  }
}

// Keeps a row's 16-bit elements packed over a reduction: without it the
// compiler holds on to their float32 values, twice the registers.
template <typename T, int NV>
__device__ __forceinline__ void StayPacked(Vec<T, kVec<T>> (&x)[NV]) {
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Words w = __builtin_bit_cast(Words, x[i]);
      asm volatile("" : "+v"(w));
      x[i] = __builtin_bit_cast(Vec<T, kVec<T>>, w);
    }
  }
}

constexpr int BlockOf(int g) { return g > 256 ? g : 256; }

// A value that all lanes of a row hold, in a scalar register where a wavefront
// has one row: above 64 vector registers a CU has one work-group of 1024
// instead of two (16,384 x 8192 bfloat16 forwards 140 us, 106).
template <int G>
__device__ __forceinline__ float RowValue(float x) {
  if constexpr (G < kWave) {
    return x;
  } else {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
  }
}

// 1 / sqrt(variance + epsilon) of a row whose values, `shift` off their mean on
// average, have a mean square of `square`. Rounding may leave a variance below
// zero; a NaN stays one, and a square past float32 gives zero, as the fused
// product does not overflow.
__device__ __forceinline__ float Rstd(float square, float shift,
                                      float epsilon) {
  const float variance = fmaf(-shift, shift, square);
  return rsqrtf((variance < 0.f ? 0.f : variance) + epsilon);
}

// The G lanes of a row take every gridDim.x-th row and keep their columns'
// weights in registers: read from the caches for every row, float32 weights of
// 16-bit rows are twice the bytes of the row and its result together (65,536 x
// 3328 bfloat16: 330 us that way, 169 this way).
template <typename T, int NV, int G, Cut kCut>
__global__ __launch_bounds__(BlockOf(G)) void NormForward(NormArgs<T> a) {
  constexpr int V = kVec<T>;
  constexpr int kRows = BlockOf(G) / G;
  constexpr int kParts = G > kWave ? G / kWave : 1;
  using At = Span<kCut, V>;
  __shared__ float part[3 * kParts];
  const int lane = threadIdx.x % G;
  const float scale = 1.f / static_cast<float>(a.dim);
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * V;
    if (c < a.dim) {
      const At s(c, a.dim);
      LoadWeights<kCut, T, V>(a.weight, a.weight_f32, s, 1.f, w[i]);
      LoadWeights<kCut, T, V>(a.bias, a.weight_f32, s, 0.f, b[i]);
    }
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows +
                     threadIdx.x / G;
       row < a.rows; row += static_cast<int64_t>(gridDim.x) * kRows) {
    const T* src = a.x + row * a.stride;
    Vec<T, V> x[NV];
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) x[i] = LoadSpan<kCut, T, V>(src, At(c, a.dim));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        const At s(c, a.dim);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sum[0] += s.Has(j) ? static_cast<float>(x[i].v[j]) : 0.f;
        }
      }
    }
    RowSum<G>(sum, part);
    StayPacked<T, NV>(x);
    const float first = RowValue<G>(sum[0] * scale);
    float left[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        const At s(c, a.dim);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d =
              s.Has(j) ? static_cast<float>(x[i].v[j]) - first : 0.f;
          left[0] += d;
          left[1] = fmaf(d, d, left[1]);
        }
      }
    }
    RowSum<G>(left, part + kParts);
    StayPacked<T, NV>(x);
    const float shift = RowValue<G>(left[0] * scale);
    const float rstd = RowValue<G>(Rstd(left[1] * scale, shift, a.epsilon));
    const float moved = RowValue<G>(-shift * rstd);
    if (lane == 0) {
      if (a.mean != nullptr) a.mean[row] = first + shift;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    T* dst = a.y + row * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        Vec<T, V> y;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xhat =
              fmaf(static_cast<float>(x[i].v[j]) - first, rstd, moved);
          y.v[j] = static_cast<T>(fmaf(xhat, w[i][j], b[i][j]));
        }
        StoreSpan<kCut, T, V>(dst, At(c, a.dim), y);
      }
    }
  }
}

// Rows longer than the registers of a work-group: three passes, the last two
// mostly from L2.
template <typename T>
__global__ __launch_bounds__(1024) void NormForwardLong(NormArgs<T> a) {
  constexpr int G = 1024;
  constexpr int V = kVec<T>;
  using At = Span<Cut::kOver, V>;
  __shared__ float part[3 * (G / kWave)];
  const float scale = 1.f / static_cast<float>(a.dim);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* src = a.x + row * a.stride;
    float sum[1] = {0.f};
    for (int c = threadIdx.x * V; c < a.dim; c += G * V) {
      const At s(c, a.dim);
      const auto x = LoadVec<T, V>(src + s.at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sum[0] += s.Has(j) ? static_cast<float>(x.v[j]) : 0.f;
      }
    }
    RowSum<G>(sum, part);
    const float first = sum[0] * scale;
    float left[2] = {0.f, 0.f};
    for (int c = threadIdx.x * V; c < a.dim; c += G * V) {
      const At s(c, a.dim);
      const auto x = LoadVec<T, V>(src + s.at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = s.Has(j) ? static_cast<float>(x.v[j]) - first : 0.f;
        left[0] += d;
        left[1] = fmaf(d, d, left[1]);
      }
    }
    RowSum<G>(left, part + G / kWave);
    const float shift = left[0] * scale;
    const float rstd = Rstd(left[1] * scale, shift, a.epsilon);
    const float moved = -shift * rstd;
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[row] = first + shift;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    T* dst = a.y + row * a.dim;
    for (int c = threadIdx.x * V; c < a.dim; c += G * V) {
      const At s(c, a.dim);
      const auto x = LoadVec<T, V>(src + s.at);
      float w[V], b[V];
      LoadWeights<Cut::kOver, T, V>(a.weight, a.weight_f32, s, 1.f, w);
      LoadWeights<Cut::kOver, T, V>(a.bias, a.weight_f32, s, 0.f, b);
      Vec<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat =
            fmaf(static_cast<float>(x.v[j]) - first, rstd, moved);
        y.v[j] = static_cast<T>(fmaf(xhat, w[j], b[j]));
      }
      StoreVec<T, V>(dst + s.at, y);
    }
  }
}

// The G lanes of a row take every gridDim.x-th row and keep their columns'
// share of the weight's and the bias's gradients in registers; at the end
// the groups of a work-group are added in LDS, in their order, and the
// work-group's sums go to `partial`. kHold: the weights stay in registers too
// (where a work-group of 1024 has 16 values a lane there is no room).
template <typename T, int NV, int G, Cut kCut, bool kStream>
__global__ __launch_bounds__(BlockOf(G)) void NormBackward(NormGradArgs<T> a) {
  constexpr int V = kVec<T>;
  constexpr int kBlock = BlockOf(G);
  constexpr int kGroups = kBlock / G;
  constexpr int kParts = G > kWave ? 2 * (G / kWave) : 1;
  constexpr bool kHold = sizeof(T) == 2 || NV * G < 4096;
  using At = Span<kCut, V>;
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
    if (kHold && c < a.dim) {
      LoadWeights<kCut, T, V>(a.weight, a.weight_f32, At(c, a.dim), 1.f, w[i]);
    }
  }
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
       row < a.rows; row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const T* px = a.x + row * a.stride;
    const T* pdy = a.dy + row * a.dy_stride;
    Vec<T, V> x[NV], dy[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        x[i] = LoadSpan<kCut, T, V, kStream>(px, At(c, a.dim));
        dy[i] = LoadSpan<kCut, T, V, kStream>(pdy, At(c, a.dim));
      }
    }
    const float mean = a.mean[row];
    const float rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        const At s(c, a.dim);
        if (!kHold) {
          LoadWeights<kCut, T, V>(a.weight, a.weight_f32, s, 1.f, w[i]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float g = static_cast<float>(dy[i].v[j]);
          const float xhat = (static_cast<float>(x[i].v[j]) - mean) * rstd;
          const float h = s.Has(j) ? g * w[i][j] : 0.f;
          sum[0] += h;
          sum[1] = fmaf(h, xhat, sum[1]);
          dw[i][j] = fmaf(g, xhat, dw[i][j]);
          db[i][j] += g;
        }
      }
    }
    RowSum<G>(sum, part + turn * kParts);
    StayPacked<T, NV>(x);
    StayPacked<T, NV>(dy);
    turn ^= 1;
    const float along1 = sum[0] * scale;
    const float alongx = sum[1] * scale;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      if (c < a.dim) {
        const At s(c, a.dim);
        if (!kHold) {
          LoadWeights<kCut, T, V>(a.weight, a.weight_f32, s, 1.f, w[i]);
        }
        Vec<T, V> dx;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xhat = (static_cast<float>(x[i].v[j]) - mean) * rstd;
          const float h = static_cast<float>(dy[i].v[j]) * w[i][j];
          dx.v[j] = static_cast<T>((h - along1 - xhat * alongx) * rstd);
        }
        StoreSpan<kCut, T, V>(a.dx + row * a.dim, s, dx);
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
        const At s(c, a.dim);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (s.Has(j)) {
            out[0][s.at + j] = dw[i][j];
            out[1][s.at + j] = db[i][j];
          }
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
        const int c = (i * G + lane) * V;
        if (c < a.dim) {
          const At s(c, a.dim);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (s.Has(j)) {
              all[group * kCols + s.at + j] = which == 0 ? dw[i][j] : db[i][j];
            }
          }
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
template <typename T>
__global__ __launch_bounds__(1024) void NormBackwardLong(NormGradArgs<T> a) {
  constexpr int G = 1024;
  constexpr int V = kVec<T>;
  constexpr int kParts = 2 * (G / kWave);
  using At = Span<Cut::kOver, V>;
  __shared__ float part[2 * kParts];
  const float scale = 1.f / static_cast<float>(a.dim);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* px = a.x + row * a.stride;
    const T* pdy = a.dy + row * a.dy_stride;
    const float mean = a.mean[row];
    const float rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f};
    for (int c = threadIdx.x * V; c < a.dim; c += G * V) {
      const At s(c, a.dim);
      const auto x = LoadVec<T, V>(px + s.at);
      const auto dy = LoadVec<T, V>(pdy + s.at);
      float w[V];
      LoadWeights<Cut::kOver, T, V>(a.weight, a.weight_f32, s, 1.f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
        const float h = s.Has(j) ? static_cast<float>(dy.v[j]) * w[j] : 0.f;
        sum[0] += h;
        sum[1] = fmaf(h, xhat, sum[1]);
      }
    }
    RowSum<G>(sum, part + turn * kParts);
    turn ^= 1;
    const float along1 = sum[0] * scale;
    const float alongx = sum[1] * scale;
    for (int c = threadIdx.x * V; c < a.dim; c += G * V) {
      const At s(c, a.dim);
      const auto x = LoadVec<T, V>(px + s.at);
      const auto dy = LoadVec<T, V>(pdy + s.at);
      float w[V];
      LoadWeights<Cut::kOver, T, V>(a.weight, a.weight_f32, s, 1.f, w);
      Vec<T, V> dx;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (static_cast<float>(x.v[j]) - mean) * rstd;
        const float h = static_cast<float>(dy.v[j]) * w[j];
        dx.v[j] = static_cast<T>((h - along1 - xhat * alongx) * rstd);
      }
      StoreVec<T, V>(a.dx + row * a.dim + s.at, dx);
    }
  }
}

// Their weight's and bias's gradients: a thread has V columns (blockIdx.x)
// and every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(256) void NormColumnsLong(NormGradArgs<T> a) {
  constexpr int V = kVec<T>;
  const int c = (blockIdx.x * 256 + threadIdx.x) * V;
  if (c >= a.dim) return;
  const Span<Cut::kOver, V> s(c, a.dim);
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const auto x = LoadVec<T, V>(a.x + row * a.stride + s.at);
    const auto dy = LoadVec<T, V>(a.dy + row * a.dy_stride + s.at);
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
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * a.dim + s.at;
  const int64_t bias = static_cast<int64_t>(gridDim.y) * a.dim;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (s.Has(j)) {
      out[j] = dw[j];
      out[bias + j] = db[j];
    }
  }
}

// Adds the work-groups' sums: kReduceColumns columns a work-group, the `parts`
// rows of sums in slices that LDS joins in their order, from column `first`
// on. Up to 1024 columns it is latency alone (6 MB at most, from L2): all of a
// thread's loads are in flight at once. 4096 columns have up to 25 MB of sums,
// 16,384 (256 parts) 34 MB, longer rows in proportion. 16 columns up to 1024
// (100 columns 3.6 us, with 32 a work-group 4.2), then 32 (4096 columns 5.8 us,
// with 16 8.9).
template <typename W, int kReduceColumns>
__global__ __launch_bounds__(1024) void NormReduce(const float* partial,
                                                   int32_t parts, int32_t dim,
                                                   int32_t first, W* dweight,
                                                   W* dbias) {
  constexpr int kSlices = 1024 / kReduceColumns;
  __shared__ float sums[kSlices][kReduceColumns + 1];
  W* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  const int col = threadIdx.x % kReduceColumns;
  const int slice = threadIdx.x / kReduceColumns;
  const int64_t begin =
      first + static_cast<int64_t>(blockIdx.x) * kReduceColumns;
  const int64_t c = begin + col;
  const float* src =
      partial + static_cast<int64_t>(blockIdx.y) * parts * dim + c;
  float s = 0.f;
  if (c < dim) {
    constexpr int kLoads = 3 * kCus / kSlices;
    for (int p = slice; p < parts; p += kLoads * kSlices) {
      float x[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = p + i * kSlices;
        x[i] = src[static_cast<int64_t>(at < parts ? at : p) * dim];
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (p + i * kSlices < parts) s += x[i];
      }
    }
  }
  sums[slice][col] = s;
  __syncthreads();
  // Joined by 4 lanes a column, a quarter of the slices each.
  if (threadIdx.x < 4 * kReduceColumns) {
    const int quarter = threadIdx.x % 4;
    const int k = threadIdx.x / 4;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < kSlices / 4; ++i) {
      s += sums[quarter * (kSlices / 4) + i][k];
    }
    s = LaneSum<4>(s);
    const int64_t to = begin + k;
    if (quarter == 0 && to < dim) out[to] = static_cast<W>(s);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// How a row is laid out over lanes: G lanes of NV vectors each, at most 16
// values a lane (their weights and, backwards, two sums stay in registers too).
// The steps are those below, each the least that holds the row: lanes past a
// row's end do nothing (262,144 x 64 bfloat16 backwards 29 us on 16 lanes, 23 on
// 8). They are not the fewest lanes everywhere: 33 to 64 vectors have a lane
// each, and 16-bit rows of 1025 to 2048 and of 4097 to 8192 columns never reach
// the second vector of {256, 2} and {1024, 2}, which costs registers alone
// (32,768 x 2048 bfloat16 47 us forwards, 5.7 TB/s, and 88 backwards, 4.6;
// 16,384 x 8192 101 and 174, 5.3 and 4.6; one vector a lane was not timed).
// G = 0 for a row that no work-group holds: in passes, 4096 rows of 20,001
// float32 take 192 us forwards and 381 backwards, 3.4 and 2.6 TB/s; in registers
// 10,000 of 16,384 take 227 and 397, 5.8 and 5.0.
struct Layout {
  int g;
  int nv;
};

Layout LayoutOf(int v, int64_t dim) {
  const int64_t n = CeilDiv(dim, v);
  const int most = 16 / v;  // vectors a lane
  return n <= 4            ? Layout{4, 1}
         : n <= 8          ? Layout{8, 1}
         : n <= 16         ? Layout{16, 1}
         : n <= 32         ? Layout{16, 2}
         : n <= 64         ? Layout{64, 1}
         : n <= 128        ? Layout{64, 2}
         : n <= 64 * most  ? Layout{64, most}
         : n <= 512        ? Layout{256, 2}
         : n <= 256 * most ? Layout{256, most}
         : n <= 2048       ? Layout{1024, 2}
         : n <= 1024 * most ? Layout{1024, most}
                            : Layout{0, 0};
}

// Work-groups of the backward pass, and so rows of partial sums: three a CU
// (65,536 x 1024 bfloat16: two 94 us, three 80, four 81; one of 1024 threads),
// each group of lanes at least one row, and no more bytes of sums written and
// read than a quarter of what the rows are (a bound on the traffic; what it
// does to the latency of a few hundred to a few thousand rows was not timed).
int64_t BackwardParts(Layout l, int type_bytes, int64_t rows) {
  const int groups = l.g == 0 ? 1 : BlockOf(l.g) / l.g;
  const int64_t most = l.g == 1024 || l.g == 0 ? kCus : 3 * kCus;
  const int64_t by_rows = CeilDiv(rows, groups);
  const int64_t by_bytes =
      std::max<int64_t>(rows * type_bytes * 3 / (4 * 16), 32);
  return std::max<int64_t>(1, std::min({most, by_rows, by_bytes}));
}

template <typename T, int NV, int G, Cut kCut>
int LaunchForward(const NormArgs<T>& a, hipStream_t stream) {
  const int64_t blocks =
      std::min<int64_t>(CeilDiv(a.rows, BlockOf(G) / G),
                        kCus * (kForwardThreads / BlockOf(G)));
  hipLaunchKernelGGL((NormForward<T, NV, G, kCut>),
                     dim3(static_cast<uint32_t>(blocks)), dim3(BlockOf(G)), 0,
                     stream, a);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T, int NV, int G, Cut kCut>
int LaunchBackward(const NormGradArgs<T>& a, int64_t parts,
                   hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(parts));
  if (a.rows * a.dim * 3 * static_cast<int64_t>(sizeof(T)) > kCacheBytes) {
    hipLaunchKernelGGL((NormBackward<T, NV, G, kCut, true>), grid,
                       dim3(BlockOf(G)), 0, stream, a);
  } else {
    hipLaunchKernelGGL((NormBackward<T, NV, G, kCut, false>), grid,
                       dim3(BlockOf(G)), 0, stream, a);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

// Returns CALL with the layout's NV and G as constants. (A row below a vector
// has one layout, 16-bit rows have at most two vectors a lane.)
#define SCEMB_LAYOUT(G_, NV_, CALL)                                        \
  if constexpr (NV_ * kVec<T> <= 16 &&                                     \
                (kCut != Cut::kPart || (G_ == 4 && NV_ == 1))) {           \
    if (l.g == G_ && l.nv == NV_) {                                        \
      constexpr int G = G_, NV = NV_;                                      \
      return CALL;                                                         \
    }                                                                      \
  }
#define SCEMB_LAYOUTS(CALL)   \
  SCEMB_LAYOUT(4, 1, CALL)    \
  SCEMB_LAYOUT(8, 1, CALL)    \
  SCEMB_LAYOUT(16, 1, CALL)   \
  SCEMB_LAYOUT(16, 2, CALL)   \
  SCEMB_LAYOUT(64, 1, CALL)   \
  SCEMB_LAYOUT(64, 2, CALL)   \
  SCEMB_LAYOUT(64, 4, CALL)   \
  SCEMB_LAYOUT(256, 2, CALL)  \
  SCEMB_LAYOUT(256, 4, CALL)  \
  SCEMB_LAYOUT(1024, 2, CALL) \
  SCEMB_LAYOUT(1024, 4, CALL)
// CALL for how rows of `dim` are cut.
#define SCEMB_CUT(CALL)                           \
  switch (CutOf(dim, kVec<T>)) {                  \
    case Cut::kWhole: {                           \
      constexpr Cut kCut = Cut::kWhole;           \
      rc = CALL;                                  \
      break;                                      \
    }                                             \
    case Cut::kOver: {                            \
      constexpr Cut kCut = Cut::kOver;            \
      rc = CALL;                                  \
      break;                                      \
    }                                             \
    default: {                                    \
      constexpr Cut kCut = Cut::kPart;            \
      rc = CALL;                                  \
    }                                             \
  }

template <typename T, Cut kCut>
int Forward(const NormArgs<T>& a, hipStream_t stream) {
  const Layout l = LayoutOf(kVec<T>, a.dim);
  SCEMB_LAYOUTS((LaunchForward<T, NV, G, kCut>(a, stream)))
  hipLaunchKernelGGL(
      NormForwardLong<T>,
      dim3(static_cast<uint32_t>(std::min(a.rows, MostGroups(1024)))),
      dim3(1024), 0, stream, a);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T, Cut kCut>
int Backward(const NormGradArgs<T>& a, Layout l, int64_t parts,
             hipStream_t stream) {
  SCEMB_LAYOUTS((LaunchBackward<T, NV, G, kCut>(a, parts, stream)))
  hipLaunchKernelGGL(
      NormBackwardLong<T>,
      dim3(static_cast<uint32_t>(std::min(a.rows, MostGroups(1024)))),
      dim3(1024), 0, stream, a);
  SCEMB_LAUNCH_CHECK();
  if (a.partial != nullptr) {
    hipLaunchKernelGGL(
        NormColumnsLong<T>,
        dim3(static_cast<uint32_t>(CeilDiv(a.dim, 256 * kVec<T>)),
             static_cast<uint32_t>(parts)),
        dim3(256), 0, stream, a);
    SCEMB_LAUNCH_CHECK();
  }
  return 0;
}
#undef SCEMB_LAYOUTS
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
  int rc = 0;
  SCEMB_CUT((Forward<T, kCut>(a, stream)))
  return rc;
}

template <typename W, int kReduceColumns>
int LaunchReduce(const float* partial, int64_t parts, int64_t dim,
                 void* dweight, void* dbias, hipStream_t stream) {
  constexpr int64_t kGroups = MostGroups(1024);
  for (int64_t first = 0; first < dim; first += kGroups * kReduceColumns) {
    const int64_t groups =
        std::min(CeilDiv(dim - first, kReduceColumns), kGroups);
    hipLaunchKernelGGL((NormReduce<W, kReduceColumns>),
                       dim3(static_cast<uint32_t>(groups), 2), dim3(1024), 0,
                       stream, partial, static_cast<int32_t>(parts),
                       static_cast<int32_t>(dim), static_cast<int32_t>(first),
                       static_cast<W*>(dweight), static_cast<W*>(dbias));
    SCEMB_LAUNCH_CHECK();
  }
  return 0;
}

template <typename W>
int RunReduce(const float* partial, int64_t parts, int64_t dim, void* dweight,
              void* dbias, hipStream_t stream) {
  return dim <= 1024 ? LaunchReduce<W, 16>(partial, parts, dim, dweight, dbias,
                                           stream)
                     : LaunchReduce<W, 32>(partial, parts, dim, dweight, dbias,
                                           stream);
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
  const Layout l = LayoutOf(kVec<T>, dim);
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
    int rc = 0;
    SCEMB_CUT((Backward<T, kCut>(a, l, parts, stream)))
    if (rc != 0) return rc;
  }
  if (a.partial == nullptr) return 0;
  const int64_t sums = rows > 0 ? parts : 0;
  return weight_f32
             ? RunReduce<float>(a.partial, sums, dim, dweight, dbias, stream)
             : RunReduce<T>(a.partial, sums, dim, dweight, dbias, stream);
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
  Arena arena(nullptr, 0);
  arena.Take<float>(
      2 * dim * BackwardParts(LayoutOf(16 / bytes, dim), bytes, rows));
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
