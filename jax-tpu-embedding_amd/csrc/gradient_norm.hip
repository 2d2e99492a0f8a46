// The norm of all values of many tensors, and what scales them down to a limit.
//
// Sums of squares are kept in 64 bits: a float32 square can be past float32's
// range on either side, and 64-bit products of two such values are exact, so
// neither a scale nor a second pass is needed. Every work-group sums a stretch
// of one tensor, and the last launch adds the work-groups' sums, both in an
// order that the sizes decide.
//
// Measured: 176M float32 values 106 us (6.6 TB/s, HBM), 79M bfloat16 ones
// clipped 88 us (read, read again from the last cache, written: 5.4 TB/s), 300
// small tensors clipped 25 us (two launches of 5 to 8 us; the rest is the host's),
// 12 of them without 7.7 us (one launch).
//
// Past 256 MB (kCacheBytes) values are read, and clipped ones written, past the
// caches: 704 MB of float32 norm 106 us, clipped 367 (through the caches 122 and
// 414), 352 MB of bfloat16 57 and 183 (62 and 203); below, through them: 200 MB of
// bfloat16 33 and 93 (past them 35 and 99), 158 MB 27 and 75 (28 and 80).
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
constexpr int kMaxTensors = 320;
struct Tensors {
  uint64_t data[kMaxTensors];  // address, and the type from bit 48 on
  uint32_t size[kMaxTensors];  // number of values
  int32_t n;
  int32_t log_step;  // values of a work-group
};
static_assert(sizeof(Tensors) <= 3904, "kernel arguments are 4096 bytes");

__device__ __forceinline__ int32_t TypeAt(uint64_t data) {
  return static_cast<int32_t>(data >> 48);
}
__device__ __forceinline__ char* AddressAt(uint64_t data) {
  return reinterpret_cast<char*>(data & ((1ull << 48) - 1));
}

// The work-group's stretch. A lane counts the stretches of neighbouring tensors.
struct Stretch {
  char* data;
  int32_t n;
  int32_t type;
};
__device__ __forceinline__ Stretch StretchOf(const Tensors& t,
                                             uint32_t group) {
  constexpr int kPer = kMaxTensors / kWave;
  const uint64_t step = 1ull << t.log_step;
  const auto stretches = [&](int i) -> uint32_t {
    return i < t.n ? static_cast<uint32_t>((t.size[i] + step - 1) >> t.log_step)
                   : 0;
  };
  const int first = LaneId() * kPer;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) mine += stretches(first + i);
  const uint32_t upto = WaveInclusiveScan(mine);
  const int who = __builtin_ctzll(__ballot(upto > group));
  uint32_t at = group - __builtin_amdgcn_readlane(upto - mine, who);
  int i = who * kPer;
  for (uint32_t n = stretches(i); at >= n; n = stretches(++i)) at -= n;
  i = __builtin_amdgcn_readfirstlane(i);
  const uint64_t begin = static_cast<uint64_t>(
      __builtin_amdgcn_readfirstlane(at)) << t.log_step;
  const uint64_t left = t.size[i] - begin;
  const int32_t type = TypeAt(t.data[i]);
  return {AddressAt(t.data[i]) + begin * (type == SCEMB_F32 ? 4 : 2),
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

// The sum over a work-group's lanes, in every one of them.
template <int kAll>
__device__ __forceinline__ double GroupSum(double x) {
  __shared__ double waves[kAll / kWave];
#pragma unroll
  for (int d = kWave / 2; d > 0; d /= 2) x += __shfl_down(x, d, kWave);
  if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = x;
  __syncthreads();
  x = waves[0];
  for (int w = 1; w < kAll / kWave; ++w) x += waves[w];
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

// A norm that is no number makes the factor none.
__device__ __forceinline__ float FactorOf(double norm, double max_norm) {
  return norm <= max_norm ? 1.f : static_cast<float>(max_norm / norm);
}

// The work-groups' sums added up by one.
template <int kAll>
__device__ __forceinline__ double SumOf(const double* parts, int32_t n) {
  double sum = 0.0;
#pragma unroll 4
  for (int32_t i = threadIdx.x; i < n; i += kAll) sum += parts[i];
  return GroupSum<kAll>(sum);
}

__global__ __launch_bounds__(kFinishThreads) void FinishNorm(
    const double* parts, int32_t n, double max_norm, float* norm,
    float* factor) {
  const double root = sqrt(SumOf<kFinishThreads>(parts, n));
  if (threadIdx.x == 0) {
    *norm = static_cast<float>(root);
    if (factor != nullptr) *factor = FactorOf(root, max_norm);
  }
}

// All of a few values by one work-group in one launch, 8 values of a lane at a
// time: two launches are 4 us each, however little they do.
constexpr int64_t kFew = 32768;
constexpr int kEach = 8;
template <typename T>
__device__ __forceinline__ double SquaresOf(const T* p, int32_t n) {
  double sum = 0.0;
  if (n >= kEach) {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int j = 0; j < kEach; j += V) {
      const auto x = LoadVec<T, V>(p + j);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double v = static_cast<double>(static_cast<float>(x.v[i]));
        sum = fma(v, v, sum);
      }
    }
  } else {
    for (int32_t j = 0; j < n; ++j) {
      const double v = static_cast<double>(static_cast<float>(p[j]));
      sum = fma(v, v, sum);
    }
  }
  return sum;
}
__global__ __launch_bounds__(kFinishThreads) void NormOfFew(
    Tensors t, double max_norm, float* norm, float* factor) {
  __shared__ int32_t first[kMaxTensors + 1];
  __shared__ int32_t scratch[kFinishThreads / kWave + 1];
  const int32_t i = threadIdx.x;
  const int32_t mine =
      i < t.n ? static_cast<int32_t>((t.size[i] + kEach - 1) / kEach) : 0;
  int32_t all;
  const int32_t before =
      BlockExclusiveScan<int32_t, kFinishThreads>(mine, scratch, &all);
  if (i < t.n) first[i] = before;
  __syncthreads();
  double sum = 0.0;
#pragma unroll 4
  for (int32_t v = threadIdx.x; v < all; v += kFinishThreads) {
    // The last tensor that begins at or before v (those of no values are not
    // given).
    int32_t lo = 0, hi = t.n;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) / 2;
      if (first[mid] <= v) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    const int32_t at = (v - first[lo]) * kEach;
    const int32_t left = static_cast<int32_t>(t.size[lo]) - at;
    const uint64_t data = t.data[lo];
    const char* p = AddressAt(data);
    if (TypeAt(data) == SCEMB_F32) {
      sum += SquaresOf(reinterpret_cast<const float*>(p) + at, left);
    } else if (TypeAt(data) == SCEMB_BF16) {
      sum += SquaresOf(reinterpret_cast<const bf16*>(p) + at, left);
    } else {
      sum += SquaresOf(reinterpret_cast<const f16*>(p) + at, left);
    }
  }
  const double root = sqrt(GroupSum<kFinishThreads>(sum));
  if (threadIdx.x == 0) {
    *norm = static_cast<float>(root);
    if (factor != nullptr) *factor = FactorOf(root, max_norm);
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

// Scales by *factor; with parts every work-group finds the factor itself (a
// launch less), and the first stores the norm.
constexpr int64_t kOwnSums = 2048;  // parts up to which that is done
template <bool kStream>
__global__ __launch_bounds__(kThreads) void ScaleTensors(
    Tensors t, const double* parts, int32_t n, double max_norm, float* norm,
    const float* factor) {
  float f;
  if (parts != nullptr) {
    const double root = sqrt(SumOf<kThreads>(parts, n));
    f = FactorOf(root, max_norm);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
      *norm = static_cast<float>(root);
    }
  } else {
    f = *factor;
  }
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

constexpr int kLogRound = 12;
static_assert(kRound == 1 << kLogRound, "values of a work-group at a time");
constexpr int kMostLog = 30;

struct Plan {
  int64_t values = 0;
  int64_t bytes = 0;
  int32_t log_step = kLogRound;
  int64_t parts = 0;  // work-groups
};
// A tensor of more than 32 bits of values goes in pieces of whole stretches.
constexpr int64_t kMostValues = 1ll << 31;

Plan PlanOf(const scemb_gradient_t* gradients, int32_t n) {
  Plan p;
  for (int32_t i = 0; i < n; ++i) {
    p.values += gradients[i].numel;
    p.bytes += gradients[i].numel * TypeBytes(gradients[i].type);
  }
  while (p.log_step < kMostLog && p.values >> p.log_step > kMostParts) {
    ++p.log_step;
  }
  for (int32_t i = 0; i < n; ++i) {
    p.parts += CeilDiv(gradients[i].numel, 1ll << p.log_step);
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
  t.log_step = plan.log_step;
  int64_t groups = 0, done = 0;
  for (int32_t i = 0; i < n; ++i) {
    const scemb_gradient_t& g = gradients[i];
    for (int64_t at = 0; at < g.numel; at += kMostValues) {
      const int64_t values = std::min(g.numel - at, kMostValues);
      const int64_t mine = CeilDiv(values, 1ll << plan.log_step);
      if (t.n == kMaxTensors || groups + mine > MostGroups(kThreads)) {
        const int rc = launch(t, groups, done);
        if (rc != 0) return rc;
        done += groups;
        groups = 0;
        t.n = 0;
      }
      t.data[t.n] = reinterpret_cast<uint64_t>(
                        static_cast<char*>(g.data) + at * TypeBytes(g.type)) |
                    static_cast<uint64_t>(g.type) << 48;
      t.size[t.n] = static_cast<uint32_t>(values);
      ++t.n;
      groups += mine;
    }
  }
  return t.n == 0 ? 0 : launch(t, groups, done);
}

int Sum(const scemb_gradient_t* gradients, int32_t n, const Plan& plan,
        double* parts, hipStream_t stream) {
  const bool past_cache = plan.bytes > kCacheBytes;
  return ForTensors(
      gradients, n, plan, [&](const Tensors& t, int64_t groups, int64_t done) {
        const dim3 grid(static_cast<uint32_t>(groups));
        if (past_cache) {
          hipLaunchKernelGGL(SquareSums<true>, grid, dim3(kThreads), 0, stream,
                             t, parts + done);
        } else {
          hipLaunchKernelGGL(SquareSums<false>, grid, dim3(kThreads), 0,
                             stream, t, parts + done);
        }
        SCEMB_LAUNCH_CHECK();
        return 0;
      });
}

int Finish(const Plan& plan, const double* parts, double max_norm, float* norm,
           float* factor, hipStream_t stream) {
  hipLaunchKernelGGL(FinishNorm, dim3(1), dim3(kFinishThreads), 0, stream,
                     parts, static_cast<int32_t>(plan.parts), max_norm, norm,
                     factor);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

// Nonzero: an error, said.
int CheckNorm(const scemb_gradient_t* gradients, int32_t n, double max_norm,
              const float* norm) {
  const int bad = CheckGradients(gradients, n);
  if (bad != 0) return bad;
  if (norm == nullptr || !(max_norm >= 0)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "gradient norm: the norm's place is missing, or max_norm is "
                "negative or no number");
  }
  return 0;
}

// The sums' places and a factor's in the workspace.
struct Space {
  double* parts;
  float* factor;
  Space(Arena* arena, const Plan& plan)
      : parts(arena->Take<double>(plan.parts)), factor(arena->Take<float>(1)) {}
};
int CheckSpace(const Arena& arena, const Plan& plan) {
  if (arena.measuring() || arena.overflow() || plan.parts > 0x7fffffff) {
    return Fail(SCEMB_ERR_WORKSPACE, "gradient norm: workspace too small");
  }
  return 0;
}

}  // namespace
}  // namespace scemb

extern "C" {

size_t scemb_gradient_norm_workspace_size(const scemb_gradient_t* gradients,
                                          int32_t num_gradients) {
  using namespace scemb;
  if (CheckGradients(gradients, num_gradients) != 0) return 0;
  Arena arena(nullptr, 0);
  Space(&arena, PlanOf(gradients, num_gradients));
  return arena.used();
}

int scemb_gradient_norm(const scemb_gradient_t* gradients,
                        int32_t num_gradients, double max_norm, float* norm,
                        float* factor, void* workspace, size_t workspace_bytes,
                        void* stream) {
  using namespace scemb;
  const int bad = CheckNorm(gradients, num_gradients, max_norm, norm);
  if (bad != 0) return bad;
  const Plan plan = PlanOf(gradients, num_gradients);
  Arena arena(workspace, workspace_bytes);
  const Space space(&arena, plan);
  const int small = CheckSpace(arena, plan);
  if (small != 0) return small;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  int32_t some = 0;  // tensors with values
  for (int32_t i = 0; i < num_gradients; ++i) some += gradients[i].numel > 0;
  if (plan.values <= kFew && some > 0 && some <= kMaxTensors) {
    return ForTensors(gradients, num_gradients, plan,
                      [&](const Tensors& t, int64_t, int64_t) {
                        hipLaunchKernelGGL(NormOfFew, dim3(1),
                                           dim3(kFinishThreads), 0, s, t,
                                           max_norm, norm, factor);
                        SCEMB_LAUNCH_CHECK();
                        return 0;
                      });
  }
  const int rc = Sum(gradients, num_gradients, plan, space.parts, s);
  if (rc != 0) return rc;
  return Finish(plan, space.parts, max_norm, norm, factor, s);
}

int scemb_clip_gradients(const scemb_gradient_t* gradients,
                         int32_t num_gradients, double max_norm, float* norm,
                         void* workspace, size_t workspace_bytes,
                         void* stream) {
  using namespace scemb;
  const int bad = CheckNorm(gradients, num_gradients, max_norm, norm);
  if (bad != 0) return bad;
  const Plan plan = PlanOf(gradients, num_gradients);
  Arena arena(workspace, workspace_bytes);
  const Space space(&arena, plan);
  const int small = CheckSpace(arena, plan);
  if (small != 0) return small;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = Sum(gradients, num_gradients, plan, space.parts, s);
  if (rc != 0) return rc;
  const bool own_sums = plan.parts > 0 && plan.parts <= kOwnSums;
  if (!own_sums) {
    rc = Finish(plan, space.parts, max_norm, norm, space.factor, s);
    if (rc != 0) return rc;
  }
  const bool past_cache = plan.bytes > kCacheBytes;
  return ForTensors(
      gradients, num_gradients, plan,
      [&](const Tensors& t, int64_t groups, int64_t done) {
        const dim3 grid(static_cast<uint32_t>(groups));
        const double* parts = own_sums ? space.parts : nullptr;
        const int32_t n = static_cast<int32_t>(plan.parts);
        float* to = done == 0 ? norm : nullptr;
        if (past_cache) {
          hipLaunchKernelGGL(ScaleTensors<true>, grid, dim3(kThreads), 0, s, t,
                             parts, n, max_norm, to, space.factor);
        } else {
          hipLaunchKernelGGL(ScaleTensors<false>, grid, dim3(kThreads), 0, s,
                             t, parts, n, max_norm, to, space.factor);
        }
        SCEMB_LAUNCH_CHECK();
        return 0;
      });
}

}  // extern "C"
