// The norm of all values of many tensors, and what scales them down to a limit.
//
// Sums of squares are kept in 64 bits: a float32 square can be past float32's
// range on either side, and 64-bit products of two such values are exact, so
// neither a scale nor a second pass is needed. Every work-group sums a stretch
// of one tensor, and the last launch adds the work-groups' sums, both in an
// order that the sizes decide.
#include <algorithm>
#include <cmath>

#include "dense.h"

namespace scemb {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;            // 16-byte vectors of a lane in flight
constexpr int64_t kRound = 4096;      // values of a work-group at a time
constexpr int64_t kMostParts = 8192;  // stretches of a call, about
constexpr int kFinishThreads = 1024;

// Tensors of a launch: what the kernel's arguments hold.
constexpr int kMaxTensors = 168;
struct Tensors {
  void* data[kMaxTensors];
  uint64_t size[kMaxTensors];   // number of values * 4 + type
  uint32_t first[kMaxTensors];  // first work-group
  int32_t n;
  int32_t rounds;  // of a work-group
};
static_assert(sizeof(Tensors) <= 3584, "kernel arguments");
static_assert(SCEMB_F32 < 4 && SCEMB_BF16 < 4 && SCEMB_F16 < 4, "two bits");

// The work-group's stretch.
struct Stretch {
  char* data;
  int32_t n;
  int32_t type;
};
__device__ __forceinline__ Stretch StretchOf(const Tensors& t,
                                             uint32_t group) {
  int i = -1;
#pragma unroll
  for (int k = 0; k < (kMaxTensors + kWave - 1) / kWave; ++k) {
    const int at = threadIdx.x % kWave + k * kWave;
    i += __popcll(__ballot(at < t.n && t.first[at] <= group));
  }
  i = __builtin_amdgcn_readfirstlane(i);
  const int64_t step = t.rounds * kRound;
  const int64_t begin = (group - t.first[i]) * step;
  const int32_t type = static_cast<int32_t>(t.size[i] & 3);
  const int64_t left = static_cast<int64_t>(t.size[i] >> 2) - begin;
  return {static_cast<char*>(t.data[i]) + begin * (type == SCEMB_F32 ? 4 : 2),
          static_cast<int32_t>(left < step ? left : step), type};
}

template <typename T, bool kStream>
__device__ __forceinline__ double SumSquares(const T* p, int32_t n) {
  constexpr int V = kVec<T>;
  double sum[2] = {0.0, 0.0};
  const auto add = [&](const Vec<T, V>& x) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double v = static_cast<double>(static_cast<float>(x.v[j]));
      sum[j % 2] = fma(v, v, sum[j % 2]);
    }
  };
  constexpr int kAll = kThreads * V;
  int32_t at = threadIdx.x * V;
  for (; at + (kUnroll - 1) * kAll + V <= n; at += kUnroll * kAll) {
    Vec<T, V> x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      x[u] = LoadVec<T, V, kStream>(p + at + u * kAll);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) add(x[u]);
  }
  for (; at < n; at += kAll) {
    if (at + V <= n) {
      add(LoadVec<T, V, kStream>(p + at));
    } else {
      for (int32_t j = at; j < n; ++j) {
        const double v = static_cast<double>(static_cast<float>(p[j]));
        sum[0] = fma(v, v, sum[0]);
      }
    }
  }
  return sum[0] + sum[1];
}

// The sum over a work-group's lanes, in thread 0.
template <int kAll>
__device__ __forceinline__ double GroupSum(double x) {
  __shared__ double waves[kAll / kWave];
#pragma unroll
  for (int d = kWave / 2; d > 0; d /= 2) x += __shfl_down(x, d, kWave);
  if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kAll / kWave; ++w) x += waves[w];
  }
  return x;
}

template <bool kStream>
__global__ __launch_bounds__(kThreads) void SquareSums(Tensors t,
                                                       double* parts) {
  const Stretch s = StretchOf(t, blockIdx.x);
  double sum;
  if (s.type == SCEMB_F32) {
    sum = SumSquares<float, kStream>(reinterpret_cast<float*>(s.data), s.n);
  } else if (s.type == SCEMB_BF16) {
    sum = SumSquares<bf16, kStream>(reinterpret_cast<bf16*>(s.data), s.n);
  } else {
    sum = SumSquares<f16, kStream>(reinterpret_cast<f16*>(s.data), s.n);
  }
  sum = GroupSum<kThreads>(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kFinishThreads) void FinishNorm(
    const double* parts, int32_t n, double max_norm, float* norm,
    float* factor) {
  double sum = 0.0;
  for (int32_t i = threadIdx.x; i < n; i += kFinishThreads) sum += parts[i];
  sum = GroupSum<kFinishThreads>(sum);
  if (threadIdx.x == 0) {
    const double root = sqrt(sum);
    *norm = static_cast<float>(root);
    // A norm that is no number makes the factor none.
    if (factor != nullptr) {
      *factor = root <= max_norm ? 1.f : static_cast<float>(max_norm / root);
    }
  }
}

template <typename T, bool kStream>
__device__ __forceinline__ void ScaleAll(T* p, int32_t n, float factor) {
  constexpr int V = kVec<T>;
  constexpr int kAll = kThreads * V;
  const auto scaled = [&](Vec<T, V> x) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x.v[j] = static_cast<T>(static_cast<float>(x.v[j]) * factor);
    }
    return x;
  };
  int32_t at = threadIdx.x * V;
  for (; at + (kUnroll - 1) * kAll + V <= n; at += kUnroll * kAll) {
    Vec<T, V> x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      x[u] = LoadVec<T, V, kStream>(p + at + u * kAll);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      StoreVec<T, V, kStream>(p + at + u * kAll, scaled(x[u]));
    }
  }
  for (; at < n; at += kAll) {
    if (at + V <= n) {
      StoreVec<T, V, kStream>(p + at, scaled(LoadVec<T, V, kStream>(p + at)));
    } else {
      for (int32_t j = at; j < n; ++j) {
        p[j] = static_cast<T>(static_cast<float>(p[j]) * factor);
      }
    }
  }
}

template <bool kStream>
__global__ __launch_bounds__(kThreads) void ScaleTensors(Tensors t,
                                                         const float* factor) {
  const float f = *factor;
  if (f == 1.f) return;
  const Stretch s = StretchOf(t, blockIdx.x);
  if (s.type == SCEMB_F32) {
    ScaleAll<float, kStream>(reinterpret_cast<float*>(s.data), s.n, f);
  } else if (s.type == SCEMB_BF16) {
    ScaleAll<bf16, kStream>(reinterpret_cast<bf16*>(s.data), s.n, f);
  } else {
    ScaleAll<f16, kStream>(reinterpret_cast<f16*>(s.data), s.n, f);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Nonzero: an error, said.
int CheckGradients(const scemb_gradient_t* gradients, int32_t n) {
  if (n < 0 || (n > 0 && gradients == nullptr)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "gradients: a negative number of them, or none given");
  }
  for (int32_t i = 0; i < n; ++i) {
    const scemb_gradient_t& g = gradients[i];
    if (g.numel < 0 || g.numel > (1ll << 60) || TypeBytes(g.type) == 0 ||
        (g.numel > 0 && g.data == nullptr)) {
      return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                  "gradients: tensor " + std::to_string(i) +
                      " is missing, of a negative size, or of a type other "
                      "than float32, bfloat16 and float16");
    }
  }
  return 0;
}

struct Plan {
  int64_t values = 0;
  int64_t bytes = 0;
  int32_t rounds = 1;  // of a work-group
  int64_t parts = 0;   // work-groups
};
Plan PlanOf(const scemb_gradient_t* gradients, int32_t n) {
  Plan p;
  for (int32_t i = 0; i < n; ++i) {
    p.values += gradients[i].numel;
    p.bytes += gradients[i].numel * TypeBytes(gradients[i].type);
  }
  p.rounds = static_cast<int32_t>(std::min<int64_t>(
      std::max<int64_t>(CeilDiv(p.values, kRound * kMostParts), 1), 1 << 16));
  for (int32_t i = 0; i < n; ++i) {
    p.parts += CeilDiv(gradients[i].numel, kRound * p.rounds);
  }
  return p;
}

// Calls launch(tensors, their work-groups, the first of them among all) until
// all tensors are done.
template <typename F>
int ForTensors(const scemb_gradient_t* gradients, int32_t n, const Plan& plan,
               const F& launch) {
  Tensors t;
  t.n = 0;
  t.rounds = plan.rounds;
  int64_t groups = 0, done = 0;
  for (int32_t i = 0; i < n; ++i) {
    const int64_t mine = CeilDiv(gradients[i].numel, kRound * plan.rounds);
    if (mine == 0) continue;
    if (t.n == kMaxTensors || groups + mine > MostGroups(kThreads)) {
      const int rc = launch(t, groups, done);
      if (rc != 0) return rc;
      done += groups;
      groups = 0;
      t.n = 0;
    }
    t.data[t.n] = gradients[i].data;
    t.size[t.n] = static_cast<uint64_t>(gradients[i].numel) << 2 |
                  static_cast<uint64_t>(gradients[i].type);
    t.first[t.n] = static_cast<uint32_t>(groups);
    ++t.n;
    groups += mine;
  }
  return t.n == 0 ? 0 : launch(t, groups, done);
}

}  // namespace
}  // namespace scemb

extern "C" {

size_t scemb_gradient_norm_workspace_size(const scemb_gradient_t* gradients,
                                          int32_t num_gradients) {
  using namespace scemb;
  if (CheckGradients(gradients, num_gradients) != 0) return 0;
  Arena arena(nullptr, 0);
  arena.Take<double>(PlanOf(gradients, num_gradients).parts);
  return arena.used();
}

int scemb_gradient_norm(const scemb_gradient_t* gradients,
                        int32_t num_gradients, double max_norm, float* norm,
                        float* factor, void* workspace, size_t workspace_bytes,
                        void* stream) {
  using namespace scemb;
  const int bad = CheckGradients(gradients, num_gradients);
  if (bad != 0) return bad;
  if (norm == nullptr || !(max_norm >= 0)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "gradient norm: the norm's place is missing, or max_norm is "
                "negative or no number");
  }
  const Plan plan = PlanOf(gradients, num_gradients);
  Arena arena(workspace, workspace_bytes);
  double* parts = arena.Take<double>(plan.parts);
  if (workspace == nullptr || arena.overflow() || plan.parts > 0x7fffffff) {
    return Fail(SCEMB_ERR_WORKSPACE, "gradient norm: workspace too small");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool past_cache = plan.bytes > kCacheBytes;
  const int rc = ForTensors(
      gradients, num_gradients, plan,
      [&](const Tensors& t, int64_t groups, int64_t done) {
        const dim3 grid(static_cast<uint32_t>(groups));
        if (past_cache) {
          hipLaunchKernelGGL(SquareSums<true>, grid, dim3(kThreads), 0, s, t,
                             parts + done);
        } else {
          hipLaunchKernelGGL(SquareSums<false>, grid, dim3(kThreads), 0, s, t,
                             parts + done);
        }
        SCEMB_LAUNCH_CHECK();
        return 0;
      });
  if (rc != 0) return rc;
  hipLaunchKernelGGL(FinishNorm, dim3(1), dim3(kFinishThreads), 0, s, parts,
                     static_cast<int32_t>(plan.parts), max_norm, norm, factor);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

int scemb_scale_gradients(const scemb_gradient_t* gradients,
                          int32_t num_gradients, const float* factor,
                          void* stream) {
  using namespace scemb;
  const int bad = CheckGradients(gradients, num_gradients);
  if (bad != 0) return bad;
  if (factor == nullptr) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "scale gradients: the factor is missing");
  }
  const Plan plan = PlanOf(gradients, num_gradients);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool past_cache = plan.bytes > kCacheBytes;
  return ForTensors(
      gradients, num_gradients, plan,
      [&](const Tensors& t, int64_t groups, int64_t) {
        const dim3 grid(static_cast<uint32_t>(groups));
        if (past_cache) {
          hipLaunchKernelGGL(ScaleTensors<true>, grid, dim3(kThreads), 0, s, t,
                             factor);
        } else {
          hipLaunchKernelGGL(ScaleTensors<false>, grid, dim3(kThreads), 0, s,
                             t, factor);
        }
        SCEMB_LAUNCH_CHECK();
        return 0;
      });
}

}  // extern "C"
