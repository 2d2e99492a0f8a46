// AdamW over many tensors at once, with moments in float32 or in 8 bits.
//
// One launch takes up to 108 tensors, whose addresses travel in the kernel
// arguments; a work-group has kStep consecutive values of one of them.
// The work is HBM-bound: 28 bytes a value with float32 throughout, 14 with
// bfloat16 gradients and moments of 8 bits, two more for a bfloat16 copy. A
// work-group has one value vector a lane and ends: with four of them in a loop,
// or read ahead of the computation, large tensors took 3% longer. Measured, step
// after step, 176M values with float32 throughout 828 us, 6.0 TB/s (797 in turn
// with other calls; a device copy moves 4.9); 79M with 8-bit moments, bfloat16
// gradients and copies 220 us, 5.8 TB/s. Where the moments are read out between
// the steps those take 245 us, the vector units busy 0.71 of the time.
//
// Moments of 8 bits are decoded, moved, used and encoded in registers. A block
// of 256 values is the four values of each lane of a wavefront, so its scale
// is a maximum over lanes. Products and sums are rounded one by one (the file
// is compiled without contraction) and codes are those of correctly rounded
// roots and quotients, so a code is a function of its block alone, whatever
// computes it. The weight's own update uses the approximate reciprocal, an ulp
// off: two ulp of the update against a correctly rounded division.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dense.h"

namespace scemb {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;                    // consecutive values of a lane
constexpr int kStep = kThreads * kPer;     // values of a work-group
constexpr int kQuant = SCEMB_ADAMW_BLOCK;  // values that share a scale
static_assert(kQuant == kWave * kPer, "a block is one step of a wavefront");

struct Tensor {
  void* param;
  const void* grad;
  uint64_t numel : 48;
  uint64_t param_bf16 : 1;
  uint64_t grad_bf16 : 1;
  uint64_t decay : 1;
  uint32_t block;  // its first block of moments
  uint32_t first;  // its first work-group
};
static_assert(sizeof(Tensor) == 32, "four words");

// Tensors of a launch: what the kernel's arguments hold, two lanes' worth at
// most (a launch of 64 small tensors takes 5 us, and so does one of 108).
template <bool kCopies>
constexpr int kMaxTensors = kCopies ? 87 : 108;

struct Moments {
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
};

// What a step multiplies with, in float32.
struct Factors {
  float grad_scale;
  float beta_1;
  float gain_1;  // 1 - beta_1
  float beta_2;
  float gain_2;  // 1 - beta_2
  float rate;    // learning_rate / (1 - beta_1^t)
  float root;    // 1 / sqrt(1 - beta_2^t)
  float epsilon;
  float keep;    // 1 - learning_rate * weight_decay
};

template <bool kCopies>
struct Tensors {
  Tensor tensors[kMaxTensors<kCopies>];
  // Every tensor's bfloat16 copy (NULL: none).
  void* copies[kCopies ? kMaxTensors<kCopies> : 1];
};

template <bool kCopies>
struct AdamArgs : Tensors<kCopies> {
  Moments moments;
  Factors factors;
  const float* rates;  // rate, root and keep made on the device, or NULL
  const float* grad_scale_ptr;
  int32_t n;
};
static_assert(sizeof(AdamArgs<false>) <= 3584 &&
                  sizeof(AdamArgs<true>) <= 3584,
              "the arguments must fit the kernel argument block");

__host__ __device__ inline void SetRates(double learning_rate, double beta_1,
                                         double beta_2, double weight_decay,
                                         int64_t step, Factors* f) {
  const double t = static_cast<double>(step);
  f->rate = static_cast<float>(learning_rate / (1.0 - pow(beta_1, t)));
  f->root = static_cast<float>(1.0 / sqrt(1.0 - pow(beta_2, t)));
  f->keep = static_cast<float>(1.0 - learning_rate * weight_decay);
}

// The same from device scalars, once a step: in every work-group of it, two
// powers in 64 bits would be three times the step's own operations.
__global__ void MakeRates(scemb_adamw_options_t o, float* rates) {
  Factors f;
  SetRates(o.learning_rate_ptr != nullptr
               ? static_cast<double>(*o.learning_rate_ptr)
               : o.learning_rate,
           o.beta_1, o.beta_2, o.weight_decay,
           o.step_ptr != nullptr ? *o.step_ptr : o.step, &f);
  if (threadIdx.x == 0) {
    rates[0] = f.rate;
    rates[1] = f.root;
    rates[2] = f.keep;
  }
}

// The lane's values, of which `count` exist (zeros past them).
template <typename T, bool kStream>
__device__ __forceinline__ void Load4(const T* p, int count,
                                      float (&x)[kPer]) {
  if (count == kPer) {
    const auto v = LoadVec<T, kPer, kStream>(p);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = static_cast<float>(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x[j] = j < count ? static_cast<float>(p[j]) : 0.f;
    }
  }
}

template <typename T, bool kStream>
__device__ __forceinline__ void Store4(T* p, int count,
                                       const float (&x)[kPer]) {
  if (count == kPer) {
    Vec<T, kPer> v;
#pragma unroll
    for (int j = 0; j < kPer; ++j) v.v[j] = static_cast<T>(x[j]);
    StoreVec<T, kPer, kStream>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j < count) p[j] = static_cast<T>(x[j]);
    }
  }
}

__device__ __forceinline__ float DecodeM(int8_t q, float scale) {
  const float x = static_cast<float>(q) * (1.f / 127.f);
  return x * fabsf(x) * scale;
}
__device__ __forceinline__ float DecodeR(uint8_t q, float scale) {
  const float x = static_cast<float>(q) * (1.f / 255.f);
  return x * x * scale;
}

// The code of x >= 0 (kLevels: 127 or 255) among values up to `scale`:
// sqrt(x / scale) * kLevels, rounded to nearest, ties to even. A scale of zero
// has only zeros below it.
template <int kLevels>
__device__ __forceinline__ float CodeExact(float x, float scale) {
  constexpr float kMost = kLevels;
  return fminf(rintf(sqrtf(x / (scale > 0.f ? scale : 1.f)) * kMost), kMost);
}

// The same code in a fifth of the instructions. With r = 1 / scale to an ulp,
// sqrt(x * r) * kLevels by the approximate root is within 2.8e-7 of the exact
// value (halves of an ulp of r and of the product's rounding, an ulp of the
// root, the last rounding), and what CodeExact rounds within 1.6e-7: at most
// 4.4e-7 * kLevels apart, or 5.6e-5 and 1.1e-4. Where the nearest half is twice
// as far away, both round alike; for the others (and for NaN), one value in
// 4000 and 2000, CodeExact decides.
template <int kLevels>
__device__ __forceinline__ float CodeFast(float x, float scale, float r) {
  constexpr float kNear = 0.5f - kLevels * 1e-6f;
  const float u = __builtin_amdgcn_sqrtf(x * r) * kLevels;
  float q = rintf(u);
  if (!(fabsf(u - q) < kNear)) q = CodeExact<kLevels>(x, scale);
  return q;
}

// Correctly rounded roots. The approximate one is an ulp off at most, and which
// of it and its neighbours is nearest follows from the signs of v - s * (its
// neighbour), which a fused multiply-add gets right (Tuckerman's test: s is
// nearest if s * (s - ulp) < v <= s * (s + ulp)). Zero, infinity and NaN fail
// both comparisons and stay. Values between zero and 2^-90, where the
// approximate root or the differences may vanish, go through sqrtf.
__device__ __forceinline__ void Roots(const float (&v)[kPer],
                                      float (&r)[kPer]) {
  uint32_t least = ~0u;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v[j]);
    least = min(least, bits - 1u);  // zero becomes the largest
    const float s = __builtin_amdgcn_sqrtf(v[j]);
    const uint32_t at = __builtin_bit_cast(uint32_t, s);
    const float below = __builtin_bit_cast(float, at - 1u);
    const float above = __builtin_bit_cast(float, at + 1u);
    float x = fmaf(-below, s, v[j]) <= 0.f ? below : s;
    x = fmaf(-above, s, v[j]) > 0.f ? above : x;
    r[j] = x;
  }
  if (least < __builtin_bit_cast(uint32_t, 0x1p-90f)) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) r[j] = sqrtf(v[j]);
  }
}

// A work-group's values of one tensor: kStep from `begin` on.
template <int kBits, typename P, typename G, bool kStream>
__device__ __forceinline__ void UpdateStep(const Tensor& t, bf16* copy,
                                           const Moments& s, const Factors& f,
                                           int64_t begin) {
  // The work-group's part is uniform: lanes only add 32-bit offsets to it.
  const int64_t slot = static_cast<int64_t>(t.block) * kQuant + begin;
  const int64_t left = static_cast<int64_t>(t.numel) - begin;
  const int here = left < kStep ? static_cast<int>(left) : kStep;
  const uint32_t own = threadIdx.x * kPer;
  // The wavefront's block of 256 values: all of its lanes go on, or none.
  const uint32_t block =
      __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (static_cast<int>(block) * kQuant >= here) return;
  const int count = min(max(here - static_cast<int>(own), 0), kPer);
  P* param = static_cast<P*>(t.param) + begin;
  const float keep = t.decay ? f.keep : 1.f;
  float p[kPer], g[kPer], m[kPer], v[kPer], r[kPer];
  Load4<P, kStream>(param + own, count, p);
  Load4<G, kStream>(static_cast<const G*>(t.grad) + begin + own, count, g);
  if constexpr (kBits == 8) {
    const auto qm =
        LoadVec<int8_t, kPer>(static_cast<const int8_t*>(s.m) + slot + own);
    const auto qv =
        LoadVec<uint8_t, kPer>(static_cast<const uint8_t*>(s.v) + slot + own);
    const float ms = s.m_scale[slot / kQuant + block];
    const float vs = s.v_scale[slot / kQuant + block];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      m[j] = DecodeM(qm.v[j], ms);
      const float root = DecodeR(qv.v[j], vs);
      v[j] = root * root;
    }
  } else {
    Load4<float, kStream>(static_cast<const float*>(s.m) + slot + own, kPer,
                          m);
    Load4<float, kStream>(static_cast<const float*>(s.v) + slot + own, kPer,
                          v);
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const float x = g[j] * f.grad_scale;
    m[j] = m[j] * f.beta_1 + x * f.gain_1;
    v[j] = v[j] * f.beta_2 + x * x * f.gain_2;
  }
  Roots(v, r);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    p[j] = p[j] * keep -
           m[j] * __builtin_amdgcn_rcpf(r[j] * f.root + f.epsilon) * f.rate;
  }
  Store4<P, kStream>(param + own, count, p);
  if (copy != nullptr) Store4<bf16, kStream>(copy + begin + own, count, p);
  if constexpr (kBits == 8) {
    // Codes past the tensor's end are zeros and stay so.
    if (count < kPer) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j >= count) m[j] = r[j] = 0.f;
      }
    }
    // The largest of values that are not negative, as bit patterns: a NaN is
    // above every number.
    uint32_t mb = 0, vb = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      mb = max(mb, __builtin_bit_cast(uint32_t, fabsf(m[j])));
      vb = max(vb, __builtin_bit_cast(uint32_t, r[j]));
    }
    const float ms = LaneReduce<LaneMaxBits, kWave>(
        __builtin_bit_cast(float, mb));
    const float vs = LaneReduce<LaneMaxBits, kWave>(
        __builtin_bit_cast(float, vb));
    // Reciprocals that do not overflow or vanish, for CodeFast. Zero and
    // non-finite scales are not among them.
    const bool fast = __builtin_amdgcn_readfirstlane(
        ms > 0x1p-100f && ms < 0x1p100f && vs > 0x1p-100f && vs < 0x1p100f);
    float cm[kPer], cv[kPer];
    if (fast) {
      const float mr = __builtin_amdgcn_rcpf(ms);
      const float vr = __builtin_amdgcn_rcpf(vs);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        cm[j] = CodeFast<127>(fabsf(m[j]), ms, mr);
        cv[j] = CodeFast<255>(r[j], vs, vr);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        cm[j] = CodeExact<127>(fabsf(m[j]), ms);
        cv[j] = CodeExact<255>(r[j], vs);
      }
    }
    Vec<int8_t, kPer> qm;
    Vec<uint8_t, kPer> qv;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      qm.v[j] = static_cast<int8_t>(copysignf(cm[j], m[j]));
      // At least 1 for r above zero, whatever its code: a float above zero
      // has bits of 1 or more.
      const uint32_t low = min(__builtin_bit_cast(uint32_t, r[j]), 1u);
      qv.v[j] = static_cast<uint8_t>(
          max(static_cast<uint32_t>(static_cast<int32_t>(cv[j])), low));
    }
    StoreVec<int8_t, kPer>(static_cast<int8_t*>(s.m) + slot + own, qm);
    StoreVec<uint8_t, kPer>(static_cast<uint8_t*>(s.v) + slot + own, qv);
    if (threadIdx.x % kWave == 0) {
      s.m_scale[slot / kQuant + block] = ms;
      s.v_scale[slot / kQuant + block] = vs;
    }
  } else {
    // Slots past the tensor's end belong to no value: their gradient was
    // read as zero, so zeros stay zeros.
    Store4<float, kStream>(static_cast<float*>(s.m) + slot + own, kPer, m);
    Store4<float, kStream>(static_cast<float*>(s.v) + slot + own, kPer, v);
  }
}

template <int kBits, bool kStream, bool kCopies>
__global__ __launch_bounds__(kThreads) void AdamUpdate(AdamArgs<kCopies> a) {
  static_assert(kMaxTensors<kCopies> <= 2 * kWave, "two tensors a lane");
  int i = -1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int at = threadIdx.x % kWave + k * kWave;
    i += __popcll(__ballot(at < a.n && a.tensors[at].first <= blockIdx.x));
  }
  i = __builtin_amdgcn_readfirstlane(i);
  const Tensor t = a.tensors[i];
  bf16* copy = kCopies ? static_cast<bf16*>(a.copies[i]) : nullptr;
  Factors f = a.factors;
  if (a.rates != nullptr) {
    f.rate = a.rates[0];
    f.root = a.rates[1];
    f.keep = a.rates[2];
  }
  if (a.grad_scale_ptr != nullptr) f.grad_scale = *a.grad_scale_ptr;
  const int64_t begin = static_cast<int64_t>(blockIdx.x - t.first) * kStep;
  if (t.param_bf16) {
    if (t.grad_bf16) {
      UpdateStep<kBits, bf16, bf16, kStream>(t, copy, a.moments, f, begin);
    } else {
      UpdateStep<kBits, bf16, float, kStream>(t, copy, a.moments, f, begin);
    }
  } else if (t.grad_bf16) {
    UpdateStep<kBits, float, bf16, kStream>(t, copy, a.moments, f, begin);
  } else {
    UpdateStep<kBits, float, float, kStream>(t, copy, a.moments, f, begin);
  }
}

// The values go past the caches: they are four times the codes, which the next
// step reads (an update of 13M values and this 67 us with them in the caches,
// 60 without).
__global__ __launch_bounds__(kThreads) void DecodeMoments(
    const int8_t* qm, const uint8_t* qv, const float* m_scale,
    const float* v_scale, int64_t begin, int64_t size, float* m, float* v) {
  const int64_t at =
      begin + (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kPer;
  if (at >= size) return;
  const auto cm = LoadVec<int8_t, kPer>(qm + at);
  const auto cv = LoadVec<uint8_t, kPer>(qv + at);
  const float ms = m_scale[at / kQuant];
  const float vs = v_scale[at / kQuant];
  Vec<float, kPer> om, ov;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    om.v[j] = DecodeM(cm.v[j], ms);
    const float root = DecodeR(cv.v[j], vs);
    ov.v[j] = root * root;
  }
  StoreVec<float, kPer, true>(m + at, om);
  StoreVec<float, kPer, true>(v + at, ov);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

int CheckState(const scemb_adamw_state_t* s) {
  if (s == nullptr || (s->bits != 8 && s->bits != 32) || s->size < 0 ||
      s->size % kQuant != 0 || s->size / kQuant > 0xffffffffll) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: state missing, bits not 8 or 32, or a size that is "
                "no multiple of the block");
  }
  if (s->size > 0 &&
      (s->m == nullptr || s->v == nullptr ||
       (s->bits == 8 && (s->m_scale == nullptr || s->v_scale == nullptr)))) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: moments or scales missing");
  }
  return 0;
}

int CheckTensor(const scemb_adamw_tensor_t& t, int32_t i) {
  const bool types = (t.param_type == SCEMB_F32 || t.param_type == SCEMB_BF16) &&
                     (t.grad_type == SCEMB_F32 || t.grad_type == SCEMB_BF16);
  if (t.numel < 0 || (t.numel > 0 && t.grad != nullptr &&
                      (!types || t.param == nullptr))) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: tensor " + std::to_string(i) +
                    ": parameter missing, a negative size, or a type other "
                    "than float32 and bfloat16");
  }
  return 0;
}

template <int kBits, bool kCopies>
int LaunchUpdate(const AdamArgs<kCopies>& a, uint32_t groups, bool past_cache,
                 hipStream_t stream) {
  if (past_cache) {
    hipLaunchKernelGGL((AdamUpdate<kBits, true, kCopies>), dim3(groups),
                       dim3(kThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((AdamUpdate<kBits, false, kCopies>), dim3(groups),
                       dim3(kThreads), 0, stream, a);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

// Launches of up to kMaxTensors tensors with a gradient each.
template <bool kCopies>
int UpdateAll(const scemb_adamw_tensor_t* tensors, int32_t num_tensors,
              const scemb_adamw_state_t& state,
              const scemb_adamw_options_t& o, bool past_cache,
              hipStream_t stream) {
  AdamArgs<kCopies> a;
  a.moments = {state.m, state.v, state.m_scale, state.v_scale};
  a.factors.grad_scale = static_cast<float>(o.grad_scale);
  a.factors.beta_1 = static_cast<float>(o.beta_1);
  a.factors.gain_1 = static_cast<float>(1.0 - o.beta_1);
  a.factors.beta_2 = static_cast<float>(o.beta_2);
  a.factors.gain_2 = static_cast<float>(1.0 - o.beta_2);
  a.factors.epsilon = static_cast<float>(o.epsilon);
  SetRates(o.learning_rate, o.beta_1, o.beta_2, o.weight_decay, o.step,
           &a.factors);
  a.grad_scale_ptr = o.grad_scale_ptr;
  a.rates = nullptr;
  if (o.learning_rate_ptr != nullptr || o.step_ptr != nullptr) {
    a.rates = state.scratch;
    hipLaunchKernelGGL(MakeRates, dim3(1), dim3(kWave), 0, stream, o,
                       state.scratch);
    SCEMB_LAUNCH_CHECK();
  }
  a.n = 0;
  constexpr int64_t kMostGroups = MostGroups(kThreads);
  uint32_t block = 0;
  int64_t groups = 0;
  const auto launch = [&]() {
    const uint32_t n = static_cast<uint32_t>(groups);
    return state.bits == 8
               ? LaunchUpdate<8, kCopies>(a, n, past_cache, stream)
               : LaunchUpdate<32, kCopies>(a, n, past_cache, stream);
  };
  for (int32_t i = 0; i < num_tensors; ++i) {
    const scemb_adamw_tensor_t& t = tensors[i];
    // A tensor of more values than a launch has threads for goes in pieces.
    for (int64_t at = 0; t.grad != nullptr && at < t.numel;
         at += kMostGroups * kStep) {
      const int64_t values = std::min(t.numel - at, kMostGroups * kStep);
      const int64_t mine = CeilDiv(values, kStep);
      if (a.n == kMaxTensors<kCopies> || groups + mine > kMostGroups) {
        const int rc = launch();
        if (rc != 0) return rc;
        a.n = 0;
        groups = 0;
      }
      Tensor& d = a.tensors[a.n];
      d.param = static_cast<char*>(t.param) + at * TypeBytes(t.param_type);
      d.grad = static_cast<const char*>(t.grad) + at * TypeBytes(t.grad_type);
      d.numel = static_cast<uint64_t>(values);
      d.param_bf16 = t.param_type == SCEMB_BF16;
      d.grad_bf16 = t.grad_type == SCEMB_BF16;
      d.decay = t.decay != 0;
      d.block = block + static_cast<uint32_t>(at / kQuant);
      d.first = static_cast<uint32_t>(groups);
      if constexpr (kCopies) {
        a.copies[a.n] = t.copy == nullptr
                            ? nullptr
                            : static_cast<char*>(t.copy) + at * sizeof(bf16);
      }
      ++a.n;
      groups += mine;
    }
    block += static_cast<uint32_t>(CeilDiv(t.numel, kQuant));
  }
  return a.n == 0 ? 0 : launch();
}

}  // namespace
}  // namespace scemb

extern "C" {

int scemb_adamw_update(const scemb_adamw_tensor_t* tensors,
                       int32_t num_tensors, const scemb_adamw_state_t* state,
                       const scemb_adamw_options_t* options, void* stream) {
  using namespace scemb;
  const int bad = CheckState(state);
  if (bad != 0) return bad;
  if (num_tensors < 0 || (num_tensors > 0 && tensors == nullptr) ||
      options == nullptr ||
      (options->step_ptr == nullptr && options->step < 1)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: tensors or options missing, or a step below 1");
  }
  if ((options->learning_rate_ptr != nullptr || options->step_ptr != nullptr) &&
      state->scratch == nullptr) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: a state without scratch takes no learning rate or "
                "step on the device");
  }
  int64_t blocks = 0, bytes = 0;
  bool copies = false;
  for (int32_t i = 0; i < num_tensors; ++i) {
    const scemb_adamw_tensor_t& t = tensors[i];
    const int rc = CheckTensor(t, i);
    if (rc != 0) return rc;
    const int64_t numel = std::min(t.numel, state->size + 1);
    blocks += CeilDiv(numel, kQuant);
    if (t.grad != nullptr) {
      bytes += numel * (TypeBytes(t.param_type) + TypeBytes(t.grad_type) +
                        (t.copy != nullptr ? 2 : 0) + state->bits / 4);
      copies = copies || t.copy != nullptr;
    }
  }
  if (blocks * kQuant > state->size) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: the state is smaller than the tensors");
  }
  // Read and written past the caches where they cannot hold it until the next
  // step: 176M float32 values 901 us through them, 828 past them; 79M with
  // 8-bit moments (whose codes stay) 250 and 220; but 4.9M values 22 and 24.
  const bool past_cache = bytes > kCacheBytes;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return copies ? UpdateAll<true>(tensors, num_tensors, *state, *options,
                                  past_cache, s)
                : UpdateAll<false>(tensors, num_tensors, *state, *options,
                                   past_cache, s);
}

int scemb_adamw_moments(const scemb_adamw_state_t* state, float* m, float* v,
                        void* stream) {
  using namespace scemb;
  const int bad = CheckState(state);
  if (bad != 0) return bad;
  if (state->size == 0) return SCEMB_OK;
  if (state->bits != 8 || m == nullptr || v == nullptr) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "adamw: moments of 32 bits are float32 already, or arrays to "
                "write are missing");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int64_t kMostGroups = MostGroups(kThreads);
  for (int64_t at = 0; at < state->size; at += kMostGroups * kStep) {
    const int64_t groups =
        std::min(CeilDiv(state->size - at, kStep), kMostGroups);
    hipLaunchKernelGGL(DecodeMoments, dim3(static_cast<uint32_t>(groups)),
                       dim3(kThreads), 0, s,
                       static_cast<const int8_t*>(state->m),
                       static_cast<const uint8_t*>(state->v), state->m_scale,
                       state->v_scale, at, state->size, m, v);
    SCEMB_LAUNCH_CHECK();
  }
  return SCEMB_OK;
}

}  // extern "C"
