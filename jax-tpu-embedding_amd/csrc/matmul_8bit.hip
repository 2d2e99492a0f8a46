// Products in 8-bit floating point (e4m3), where 128 values share a scale.
//
// A scale is a power of two, 2^e with the least e that leaves no value of the
// block above 448, the largest code: dividing by it is exact, so a code is the
// value rounded once. The products are bfloat16's (E4m3 in tiles.h says why): a
// code times its power of two is one conversion, two codes an instruction. The
// exponents are kept in 32 bits so that a lane loads its row's with one
// instruction. Sums are float32.
//
// Codes are laid out by row and by output column, 128 of the sum's index one
// after another (zeros behind the last), so both operands of the product are
// panels along the depth and a step of the product is a block: a scale for each
// row and one for 128 columns.
//
// Measured, bfloat16 rows, 64 experts with 131,072 rows, 1024 x 4096: 1130 us, 84
// of them the rows' quantisation (HBM, 4.8 TB/s) and the rest the product (1.05
// PFLOP/s; by the 8-bit instructions, which cut products, 840 in all), 3750 where
// every row's powers are past bfloat16; 32 rows: 16 us, the weights at HBM's rate
// after 5 us of a first launch; 20,011 rows, 3328 x 1000 float16 155 us, 36 of them
// the quantisation (115 by the 8-bit ones), 1 to 64 of them 19.
#include <algorithm>

#include "tiles.h"

namespace scemb {
namespace {

constexpr int kBlock = SCEMB_BLOCK_8BIT;
constexpr int32_t kLeast = -126;  // exponent
constexpr int32_t kBias = 127;
constexpr uint8_t kNan8 = 0x7f;

// The exponent of a block with the largest magnitude `top`.
__device__ __forceinline__ int32_t ExponentOf(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  // top = 1.m * 2^x is within 448 * 2^e = 1.75 * 2^(8 + e).
  const int32_t x = static_cast<int32_t>(bits >> 23) - 127;
  return max(x - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), kLeast);
}

// Codes of two values times 2^-e, in the low 16 bits.
__device__ __forceinline__ uint32_t Codes(float a, float b) {
  return static_cast<uint32_t>(
             __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

__device__ __forceinline__ float PowerOf(int32_t e) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(e + kBias) << 23);
}

// ---------------------------------------------------------------------------
// Rows: 16 lanes a block of 128 columns.
// ---------------------------------------------------------------------------

constexpr int kRowThreads = 256;
constexpr int kRowBlocks = kRowThreads / 16;  // of a work-group, in one column

template <typename T>
__global__ __launch_bounds__(kRowThreads) void QuantizeRows(
    const T* x, int64_t stride, int32_t rows, int32_t dim, int32_t padded,
    const int32_t* offsets, int32_t experts, uint8_t* codes,
    int32_t* exponents) {
  const int32_t row = blockIdx.x * kRowBlocks + threadIdx.x / 16;
  if (row >= rows) return;
  if (offsets != nullptr && (row < offsets[0] || row >= offsets[experts])) {
    return;
  }
  const T* from = x + row * stride;
  for (int32_t block = blockIdx.y; block < padded / kBlock;
       block += gridDim.y) {
    const int32_t at = block * kBlock + threadIdx.x % 16 * 8;
    float v[8];
    if (at + 8 <= dim) {
      constexpr int V = kVec<T>;
#pragma unroll
      for (int j = 0; j < 8; j += V) {
        const auto w = LoadVec<T, V>(from + at + j);
#pragma unroll
        for (int i = 0; i < V; ++i) v[j + i] = static_cast<float>(w.v[i]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = at + j < dim ? static_cast<float>(from[at + j]) : 0.f;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = LaneMaxBits::Of(top, fabsf(v[j]));
    top = LaneReduce<LaneMaxBits, 16>(top);
    const bool finite = top < __builtin_inff();
    const int32_t e = ExponentOf(top);
    const float scale = PowerOf(-e);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = finite ? Codes(v[2 * j] * scale, v[2 * j + 1] * scale)
                    : kNan8 * 0x101u;
    }
    *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(row) * padded + at) =
        uint2{c[0] | c[1] << 16, c[2] | c[3] << 16};
    if (threadIdx.x % 16 == 0) {
      // Zeros are zeros with any power: one that bfloat16 holds.
      exponents[static_cast<int64_t>(block) * rows + row] =
          finite && top > 0.f ? e + kBias : kBias;
    }
  }
}

// ---------------------------------------------------------------------------
// Weights: a work-group a block of 128 x 128.
// ---------------------------------------------------------------------------

constexpr int kWeightThreads = 256;
constexpr int kPitch = kBlock + 16;  // of a column's codes in LDS

// kByOuter: outer is the contiguous dimension.
template <typename T, bool kByOuter>
__global__ __launch_bounds__(kWeightThreads) void QuantizeWeights(
    const T* w, int64_t expert_stride, int64_t stride, int32_t inner,
    int32_t outer, int32_t padded, uint8_t* codes, int32_t* exponents) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock * kPitch];
  __shared__ float tops[kWeightThreads / kWave];
  const int32_t down = padded / kBlock;
  const int32_t across = (outer + kBlock - 1) / kBlock;
  const int32_t kb = blockIdx.x % down;
  const int32_t nb = blockIdx.x / down % across;
  const int64_t e = blockIdx.x / down / across;
  w += e * expert_stride;
  // A thread has one index of the contiguous dimension and half of the other's.
  const int32_t fast = threadIdx.x % kBlock;
  const int32_t slow = threadIdx.x / kBlock;
  constexpr int kEach = kBlock * kBlock / kWeightThreads;
  float v[kEach];
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int32_t other = slow + j * (kWeightThreads / kBlock);
    const int32_t k = kb * kBlock + (kByOuter ? other : fast);
    const int32_t n = nb * kBlock + (kByOuter ? fast : other);
    v[j] = k < inner && n < outer
               ? static_cast<float>(kByOuter ? w[k * stride + n]
                                             : w[n * stride + k])
               : 0.f;
    top = LaneMaxBits::Of(top, fabsf(v[j]));
  }
  top = LaneReduce<LaneMaxBits, kWave>(top);
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWeightThreads / kWave; ++i) {
    top = LaneMaxBits::Of(top, tops[i]);
  }
  const bool finite = top < __builtin_inff();
  const int32_t exponent = ExponentOf(top);
  const float scale = PowerOf(-exponent);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int32_t other = slow + j * (kWeightThreads / kBlock);
    const int32_t k = kByOuter ? other : fast;
    const int32_t n = kByOuter ? fast : other;
    tile[n * kPitch + k] =
        finite ? static_cast<uint8_t>(Codes(v[j] * scale, 0.f)) : kNan8;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBlock * kBlock / 16; i += kWeightThreads) {
    const int32_t n = i / (kBlock / 16), part = i % (kBlock / 16) * 16;
    if (nb * kBlock + n < outer) {
      *reinterpret_cast<U32x4*>(
          codes + (e * outer + nb * kBlock + n) * padded + kb * kBlock + part) =
          *reinterpret_cast<const U32x4*>(tile + n * kPitch + part);
    }
  }
  if (threadIdx.x == 0) {
    exponents[(e * across + nb) * down + kb] =
        finite ? exponent + kBias : kBias;
  }
}

// ---------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------

// The scales of a wavefront's rows and of its columns, a step ahead. A code times
// its power of two is past bfloat16 near the ends of float32 (256 * 2^120, 2^-9 *
// 2^-126): what the columns' power is out of, the rows' make up for; `lost` says
// that the rows' were out of it themselves, in any lane and step.
template <int kFragM>
struct Scales {
  const int32_t* a_from;  // of the tile's first row in the next block
  int64_t a_step;
  const int32_t* b_from;
  int32_t row[kFragM];
  int32_t a[kFragM];
  int32_t b;
  bool lost;
  int32_t next_a[kFragM];
  int32_t next_b;

  __device__ __forceinline__ void Load() {
#pragma unroll
    for (int i = 0; i < kFragM; ++i) next_a[i] = a_from[row[i]];
    next_b = *b_from;
    a_from += a_step;
    ++b_from;
  }
  __device__ __forceinline__ void Take() {
    b = min(max(next_b, kLeastHeld), kMostHeld);
    bool held = true;
#pragma unroll
    for (int i = 0; i < kFragM; ++i) {
      a[i] = next_a[i] + next_b - b;
      held = held && a[i] >= kLeastHeld && a[i] <= kMostHeld;
    }
    lost = lost || __builtin_amdgcn_ballot_w64(!held) != 0;
  }
};

// The tile's results of a wavefront whose scales were lost: the codes' own
// products, and a block's sum times its powers of two. From memory, 32 rows after
// another: it is rare, and needs no registers that the other way has use for.
template <typename C, typename Out>
__device__ __forceinline__ void StoreUnscaled(
    const uint8_t* x, const int32_t* x_exponents, int64_t x_step, int m,
    const uint8_t* w, const int32_t* w_exponents, int n, int32_t padded, Out* y,
    int64_t columns, char* lds) {
  using R = RowsOut<Out, C::kFragN>;
  const int lane = threadIdx.x % kWave;
  const int part = lane / 32 * 16;
  lds += __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * R::kBytes;
#pragma unroll 1
  for (int i = 0; i < C::kFragM; ++i) {
    const int row = C::WaveM() + i * 32;
    if (row >= m) break;
    const int32_t mine = min(row + lane % 32, m - 1);
    F32x16 acc[C::kFragN] = {};
#pragma unroll 1
    for (int32_t block = 0; block < padded / kBlock; ++block) {
      const int power = x_exponents[block * x_step + mine] +
                        w_exponents[block] - 2 * kBias;
#pragma unroll
      for (int j = 0; j < C::kFragN; ++j) {
        const int32_t column = min(C::WaveN() + j * 32 + lane % 32, n - 1);
        F32x16 sum = {};
#pragma unroll
        for (int k = 0; k < kBlock; k += 32) {
          const int64_t at = block * kBlock + k + part;
          const Wide a = Widen(*reinterpret_cast<const U32x4*>(
              x + static_cast<int64_t>(mine) * padded + at), kUnscaled);
          const Wide b = Widen(*reinterpret_cast<const U32x4*>(
              w + static_cast<int64_t>(column) * padded + at), kUnscaled);
          MultiplyAdd<bf16>(b.v[0], a.v[0], &sum);
          MultiplyAdd<bf16>(b.v[1], a.v[1], &sum);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          acc[j][k] += __builtin_ldexpf(sum[k], power);
        }
      }
    }
    R::Store(acc, lds, y + row * columns + C::WaveN(), columns, m - row,
             n - C::WaveN());
  }
}

template <typename C, typename Out>
__global__ __launch_bounds__(C::kThreads, 2) void Product8(
    const uint8_t* x, const int32_t* x_exponents, int32_t rows, int32_t padded,
    const uint8_t* w, const int32_t* w_exponents, int32_t columns,
    const int32_t* offsets, int32_t experts, Out* y, TileGrid grid) {
  __shared__ __attribute__((aligned(16))) char lds0[C::kLds];
  __shared__ __attribute__((aligned(16))) char lds1[C::kLds];
  int32_t tile, column;
  if (!grid.Tile(blockIdx.x, &tile, &column)) return;
  const RowTile t = FindRowTile(offsets, experts, rows, tile, C::kM);
  if (t.segment < 0) return;
  column *= C::kN;
  const int m = min(t.end - t.row, C::kM);
  const int n = min(columns - column, C::kN);
  C c;
  Scales<C::kFragM> scales;
  scales.a_from = x_exponents + t.row;
  scales.a_step = rows;
#pragma unroll
  for (int i = 0; i < C::kFragM; ++i) {
    scales.row[i] =
        min(C::WaveM() + i * 32 + static_cast<int>(threadIdx.x % 32), m - 1);
  }
  const int32_t across = (columns + kBlock - 1) / kBlock;
  // A wavefront past the last column has some block.
  const int32_t block = min((column + C::WaveN()) / kBlock, across - 1);
  scales.b_from =
      w_exponents + (static_cast<int64_t>(t.segment) * across + block) *
                        (padded / kBlock);
  using E = typename C::T;
  const E* a = reinterpret_cast<const E*>(x) +
               static_cast<int64_t>(t.row) * padded;
  const E* b = reinterpret_cast<const E*>(w) +
               (static_cast<int64_t>(t.segment) * columns + column) * padded;
  scales.lost = false;
  c.Run(a, padded, m, padded, b, padded, n, padded,
        t.segment < experts ? padded : 0, lds0,
        lds1, scales);
  Out* to = y + static_cast<int64_t>(t.row) * columns + column;
  if (__builtin_expect(scales.lost, 0)) {
    StoreUnscaled<C>(reinterpret_cast<const uint8_t*>(a),
                     x_exponents + t.row, rows, m,
                     reinterpret_cast<const uint8_t*>(b),
                     w_exponents + (static_cast<int64_t>(t.segment) * across +
                                    block) * (padded / kBlock),
                     n, padded, to, columns, lds0);
  } else {
    c.Store(to, columns, m, n, lds0);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

int64_t PaddedOf(int64_t inner) { return RoundUp(inner, kBlock); }

// Nonzero: an error, said.
int CheckSizes(int64_t rows, int64_t inner, int64_t outer, int32_t experts) {
  constexpr int64_t kMost = 0x7fffffff - 65536;
  if (rows < 0 || rows > kMost || inner < 1 || inner > SCEMB_MAX_INNER_8BIT ||
      outer < 1 || outer > kMost || experts < 1 ||
      experts > SCEMB_MAX_EXPERTS) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "8-bit product: rows or outer outside [1, 2^31 - 2^16) (rows "
                "may be 0), inner outside [1, 2^22], or experts outside [1, "
                "1024]");
  }
  return 0;
}

template <typename Out>
struct Call8 {
  const uint8_t* x;
  const int32_t* x_exponents;
  int64_t rows;
  int64_t padded;
  const uint8_t* w;
  const int32_t* w_exponents;
  int64_t columns;
  const int32_t* offsets;
  int32_t experts;
  Out* y;
  hipStream_t stream;

  template <typename C>
  int Launch() const {
    const TileGrid grid(rows / C::kM + experts + kNone,
                        CeilDiv(columns, C::kN));
    if (grid.Groups() > MostGroups(C::kThreads)) {
      return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                  "8-bit product: more tiles than a launch takes");
    }
    hipLaunchKernelGGL((Product8<C, Out>), dim3(grid.Groups()),
                       dim3(C::kThreads), 0, stream, x, x_exponents,
                       static_cast<int32_t>(rows),
                       static_cast<int32_t>(padded), w, w_exponents,
                       static_cast<int32_t>(columns), offsets, experts, y,
                       grid);
    SCEMB_LAUNCH_CHECK();
    return 0;
  }

  int Run() const {
    constexpr Along kDepth = Along::kDepth;
    if (WorthSmall(rows, columns, experts)) {
      return Launch<SmallTile<E4m3, kDepth, kDepth, true>>();
    }
    if (rows >= 256ll * experts && WorthLarge(rows, columns)) {
      return Launch<LargeTile<E4m3, kDepth, kDepth>>();
    }
    return Launch<MiddleTile<E4m3, kDepth, kDepth, true>>();
  }
};

template <typename T>
int RunRows(const void* x, int64_t stride, int64_t rows, int64_t dim,
            const int32_t* offsets, int32_t experts, uint8_t* codes,
            int32_t* exponents, hipStream_t stream) {
  const int64_t padded = PaddedOf(dim);
  // Work-groups of 16 rows, and as many columns of blocks at once as a launch
  // takes.
  const int64_t down = CeilDiv(rows, kRowBlocks);
  const int64_t across = std::min<int64_t>(padded / kBlock, 65535);
  if (down > MostGroups(kRowThreads)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "8-bit product: more rows than a launch takes");
  }
  const dim3 grid(
      static_cast<uint32_t>(down),
      static_cast<uint32_t>(std::max<int64_t>(
          std::min(across, MostGroups(kRowThreads) / down), 1)));
  hipLaunchKernelGGL(QuantizeRows<T>, grid, dim3(kRowThreads), 0, stream,
                     static_cast<const T*>(x), stride,
                     static_cast<int32_t>(rows), static_cast<int32_t>(dim),
                     static_cast<int32_t>(padded), offsets, experts, codes,
                     exponents);
  SCEMB_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int RunWeights(const void* w, int64_t expert_stride, int64_t inner_stride,
               int64_t outer_stride, int64_t inner, int64_t outer,
               int32_t experts, uint8_t* codes, int32_t* exponents,
               hipStream_t stream) {
  const int64_t padded = PaddedOf(inner);
  const int64_t groups =
      padded / kBlock * CeilDiv(outer, kBlock) * experts;
  if (groups > MostGroups(kWeightThreads)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "8-bit weights: more blocks than a launch takes");
  }
  const dim3 grid(static_cast<uint32_t>(groups));
  const T* from = static_cast<const T*>(w);
  const int32_t i = static_cast<int32_t>(inner);
  const int32_t o = static_cast<int32_t>(outer);
  const int32_t p = static_cast<int32_t>(padded);
  if (outer_stride == 1) {
    hipLaunchKernelGGL((QuantizeWeights<T, true>), grid, dim3(kWeightThreads),
                       0, stream, from, expert_stride, inner_stride, i, o, p,
                       codes, exponents);
  } else {
    hipLaunchKernelGGL((QuantizeWeights<T, false>), grid, dim3(kWeightThreads),
                       0, stream, from, expert_stride, outer_stride, i, o, p,
                       codes, exponents);
  }
  SCEMB_LAUNCH_CHECK();
  return 0;
}

}  // namespace
}  // namespace scemb

extern "C" {

int scemb_quantize_weights(const void* weights, int32_t type,
                           int64_t expert_stride, int64_t inner_stride,
                           int64_t outer_stride, int64_t inner, int64_t outer,
                           int32_t num_experts, uint8_t* codes,
                           int32_t* exponents, void* stream) {
  using namespace scemb;
  const int bad = CheckSizes(0, inner, outer, num_experts);
  if (bad != 0) return bad;
  if (TypeBytes(type) == 0 || weights == nullptr || codes == nullptr ||
      exponents == nullptr || expert_stride < 0 || inner_stride < 0 ||
      outer_stride < 0 || (inner_stride != 1 && outer_stride != 1)) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "8-bit weights: an operand is missing, not float32, bfloat16 "
                "or float16, or contiguous in neither inner nor outer");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto zero) {
    return RunWeights<decltype(zero)>(weights, expert_stride, inner_stride,
                                      outer_stride, inner, outer, num_experts,
                                      codes, exponents, s);
  };
  return type == SCEMB_F32    ? run(float{})
         : type == SCEMB_BF16 ? run(bf16{})
                              : run(f16{});
}

size_t scemb_matmul_8bit_workspace_size(int64_t num_rows, int64_t inner) {
  using namespace scemb;
  if (CheckSizes(num_rows, inner, 1, 1) != 0) return 0;
  Arena arena(nullptr, 0);
  arena.Take<uint8_t>(num_rows * PaddedOf(inner));
  arena.Take<int32_t>(num_rows * (PaddedOf(inner) / kBlock));
  return arena.used();
}

int scemb_matmul_8bit(const void* rows, int32_t type, int64_t rows_stride,
                      int64_t num_rows, int64_t inner, int64_t outer,
                      const uint8_t* codes, const int32_t* exponents,
                      const int32_t* offsets, int32_t num_experts, void* y,
                      void* workspace, size_t workspace_bytes, void* stream) {
  using namespace scemb;
  const int bad = CheckSizes(num_rows, inner, outer, num_experts);
  if (bad != 0) return bad;
  if (num_rows == 0) return SCEMB_OK;
  if (TypeBytes(type) == 0 || rows == nullptr || rows_stride < 0 ||
      codes == nullptr || exponents == nullptr || y == nullptr ||
      (offsets == nullptr && num_experts != 1) ||
      reinterpret_cast<uintptr_t>(codes) % 16 != 0) {
    return Fail(SCEMB_ERR_INVALID_ARGUMENT,
                "8-bit product: an operand is missing, rows that are not "
                "float32, bfloat16 or float16, a negative stride, codes that "
                "are not aligned to 16 bytes, or experts without offsets");
  }
  Arena arena(workspace, workspace_bytes);
  uint8_t* x = arena.Take<uint8_t>(num_rows * PaddedOf(inner));
  int32_t* e = arena.Take<int32_t>(num_rows * (PaddedOf(inner) / kBlock));
  if (workspace == nullptr || arena.overflow() ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return Fail(SCEMB_ERR_WORKSPACE,
                "8-bit product: workspace too small or not aligned to 16 "
                "bytes");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    const int rc = RunRows<T>(rows, rows_stride, num_rows, inner, offsets,
                              num_experts, x, e, s);
    if (rc != 0) return rc;
    const Call8<T> call = {x, e, num_rows, PaddedOf(inner), codes, exponents,
                           outer, offsets, num_experts, static_cast<T*>(y), s};
    return call.Run();
  };
  return type == SCEMB_F32    ? run(float{})
         : type == SCEMB_BF16 ? run(bf16{})
                              : run(f16{});
}

}  // extern "C"
