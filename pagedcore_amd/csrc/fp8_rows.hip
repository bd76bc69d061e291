// Rows rounded to 8 bits for the 8-bit projections: e4m3 values with a power of two per block of
// 128 columns (fp8_device.h), from fp16 rows and as the output of the residual add + RMSNorm.
//
// The reference has fp16 only; these take the place of the fp16 tensors that its projections read
// (src/pagedcore/dense.py:17-21 and 91-104 via src/pagedcore/decoder.py:156-199). The norm's output is rounded once,
// from fp32 to 8 bits: the fp16 tensors in between (and their roundings) do not exist here.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "fp8_device.h"
#include "pagedcore_hip.h"
#include "pc_internal.h"

namespace {

using namespace fp8_device;
using pc_internal::aligned;
using pc_internal::check_launch;
using pc_internal::ok;
using pc_internal::set_error;

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kMaxWidth = 1 << 22;
constexpr int kMaxNormRows = (1 << 24) - 1;     // a workgroup each: a grid's threads stay within 32 bits
constexpr int kMaxQuantizeBlocks = 1 << 29;    // eight threads each
constexpr int kNormMaxChunks = 4;  // rows of up to 4 * 256 * 8 = 8192

// Eight columns of a row per lane, the 16 lanes of a wave row one block: its scale, and the values.
__device__ __forceinline__ uint2_t round8(const float (&y)[8], int& scale) {
  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = fmaxf(largest, finite_magnitude(y[i]));
  scale = scale_of(max16(largest));
  const float inverse = inverse_of(scale);
  return uint2_t{pack4(y[0] * inverse, y[1] * inverse, y[2] * inverse, y[3] * inverse),
                 pack4(y[4] * inverse, y[5] * inverse, y[6] * inverse, y[7] * inverse)};
}

// One block of 128 columns per 16 lanes and turn, kTurns turns with every load before the first use. What bounds
// it: HBM (2 bytes read, 1 written per element). 2048 x 5632: 8.3 us, 4160 GB/s (loads that allocate in the caches 9.3, one
// turn 9.4, four 9.5).
constexpr int kTurns = 2;
__global__ __launch_bounds__(kThreads) void quantize_fp8_kernel(uint8_t* values, uint8_t* scales, const _Float16* x,
                                                                int64_t x_stride, uint32_t blocks, uint32_t row_blocks,
                                                                int32_t width) {
  half8_t v[kTurns];
  uint32_t row[kTurns], in_row[kTurns];
  const uint32_t first = blockIdx.x * (kTurns * kThreads / 16) + threadIdx.x / 16;
  auto column = [&](int i) { return static_cast<int>(in_row[i] * kBlock + 8 * (threadIdx.x % 16)); };
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const uint32_t block = min(first + i * (kThreads / 16), blocks - 1);  // past the end: the last again, not stored
    row[i] = block / row_blocks;
    in_row[i] = block - row[i] * row_blocks;
    v[i] = half8_t{};
    if (column(i) < width) v[i] = __builtin_nontemporal_load(reinterpret_cast<const half8_t*>(x + row[i] * x_stride + column(i)));
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(v[i][e]);
    int scale;
    const uint2_t packed = round8(y, scale);
    if (first + i * (kThreads / 16) >= blocks) return;
    if (column(i) < width) *reinterpret_cast<uint2_t*>(values + static_cast<int64_t>(row[i]) * width + column(i)) = packed;
    if (threadIdx.x % 16 == 0) scales[static_cast<int64_t>(row[i]) * scale_stride(width) + in_row[i]] = static_cast<uint8_t>(scale);
  }
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(q[0]) + __uint_as_float(q[1]);
  x = add_dpp<0x128>(x);  // rotations by 8, 4, 2 and 1 within 16 lanes
  x = add_dpp<0x124>(x);
  x = add_dpp<0x122>(x);
  return add_dpp<0x121>(x);
}

constexpr int kNoDelta = -1, kHalfDelta = 0;  // else: that many fp32 partial sums
constexpr int kAnySplits = 64;                // a count without its own instance (`splits`)

// One workgroup per row, eight columns per thread and chunk. The sum of the residual stream is an
// fp16 row (the next layer's residual), rounded as the fp16 form rounds it; the mean of squares and the
// norm are fp32. What bounds it: at decode sizes one round trip of memory (every load is issued
// before the first wait; 1, 2, 4 and 8 splits have instances of their own for that), at
// prompt sizes HBM. FULL: every thread has all its chunks (no branch around the loads). 1 row of 2048 and 4 splits: 2.1 us
// (a launch alone is 1.9), 128 rows and 8 splits 3.6 (2660 GB/s from the caches; 4.0 from HBM), 2048 rows and an fp16 delta
// 6.9 (4270 GB/s; 8.2 where the loads allocate in the caches, which partial sums, read where they were just written, do
// better with).
template <int CHUNKS, bool FULL, int DELTA>
__global__ __launch_bounds__(kThreads) void add_rms_norm_fp8_kernel(const _Float16* hidden, const void* delta,
                                                                    int64_t parts_stride, const _Float16* weight,
                                                                    _Float16* hidden_out, uint8_t* values, int32_t splits,
                                                                    int32_t width, uint8_t* scales, float eps) {
  constexpr int kParts = DELTA > 0 && DELTA < kAnySplits ? DELTA : 1;
  __shared__ float wave_sums[kThreads / 64];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * width;
  const int tid = threadIdx.x;
  auto column = [&](int c) { return 8 * (tid + c * kThreads); };
  auto mine = [&](int c) { return FULL || column(c) < width; };
  half8_t sum[CHUNKS], wt[CHUNKS], d[CHUNKS];
  float4_t lo[CHUNKS][kParts], hi[CHUNKS][kParts];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    sum[c] = wt[c] = half8_t{};
    if (!mine(c)) continue;
    const int64_t at = base + column(c);
    if constexpr (DELTA == kHalfDelta) d[c] = __builtin_nontemporal_load(reinterpret_cast<const half8_t*>(static_cast<const _Float16*>(delta) + at));
    if constexpr (DELTA > 0) {
#pragma unroll
      for (int s = 0; s < kParts; ++s) {
        lo[c][s] = *reinterpret_cast<const float4_t*>(static_cast<const float*>(delta) + at + s * parts_stride);
        hi[c][s] = *reinterpret_cast<const float4_t*>(static_cast<const float*>(delta) + at + s * parts_stride + 4);
      }
    }
    if constexpr (DELTA == kHalfDelta) sum[c] = __builtin_nontemporal_load(reinterpret_cast<const half8_t*>(hidden + at));
    else sum[c] = *reinterpret_cast<const half8_t*>(hidden + at);
    wt[c] = *reinterpret_cast<const half8_t*>(weight + column(c));
  }
  float squares = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (!mine(c)) continue;
    const int64_t at = base + column(c);
    if constexpr (DELTA > 0) {  // added in split order
#pragma unroll
      for (int s = 1; s < kParts; ++s) {
        lo[c][0] += lo[c][s];
        hi[c][0] += hi[c][s];
      }
      if constexpr (DELTA == kAnySplits) {
        const float* parts = static_cast<const float*>(delta) + at;
#pragma unroll 4
        for (int s = 1; s < splits; ++s) {
          lo[c][0] += *reinterpret_cast<const float4_t*>(parts + s * parts_stride);
          hi[c][0] += *reinterpret_cast<const float4_t*>(parts + s * parts_stride + 4);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[c][i] = static_cast<_Float16>(lo[c][0][i]);
        d[c][i + 4] = static_cast<_Float16>(hi[c][0][i]);
      }
    }
    if constexpr (DELTA != kNoDelta) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[c][i] = static_cast<_Float16>(static_cast<float>(sum[c][i]) + static_cast<float>(d[c][i]));
    }
    if (DELTA != kNoDelta || hidden_out != nullptr) *reinterpret_cast<half8_t*>(hidden_out + at) = sum[c];
#pragma unroll
    for (int i = 0; i < 8; ++i) squares += static_cast<float>(sum[c][i]) * static_cast<float>(sum[c][i]);
  }
  squares = wave_sum(squares);
  if ((tid & 63) == 0) wave_sums[tid >> 6] = squares;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) total += wave_sums[w];
  const float norm = 1.0f / sqrtf(total / static_cast<float>(width) + eps);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // the first product is exact in fp32
      y[i] = static_cast<float>(sum[c][i]) * static_cast<float>(wt[c][i]) * norm;
    }
    if (!FULL && !mine(c)) {  // a NaN norm times a column past the row is not the block's
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.0f;
    }
    int scale;
    const uint2_t packed = round8(y, scale);
    if (!mine(c)) continue;
    *reinterpret_cast<uint2_t*>(values + base + column(c)) = packed;
    if (tid % 16 == 0) {
      scales[static_cast<int64_t>(blockIdx.x) * scale_stride(width) + column(c) / kBlock] = static_cast<uint8_t>(scale);
    }
  }
}

int add_rms_norm_fp8(void* values, void* scales, void* hidden_out, const void* hidden, const void* delta,
                     const float* parts, int32_t splits, const void* weight, int64_t rows, int32_t width, float eps,
                     void* stream) {
  if (rows < 0 || rows > kMaxNormRows) return set_error(PC_ERR_ARGUMENT, "rows %lld out of range", static_cast<long long>(rows));
  if (width < 16 || width % 16 != 0 || width > 8 * kThreads * kNormMaxChunks) {
    return set_error(PC_ERR_ARGUMENT, "width %d must be a multiple of 16 in [16, %d]", width, 8 * kThreads * kNormMaxChunks);
  }
  if (rows == 0) return ok();  // nothing to read or write (empty buffers may be null)
  if (!values || !scales || !hidden || !weight) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if ((delta || parts) && !hidden_out) return set_error(PC_ERR_ARGUMENT, "a delta needs hidden_out for the sum");
  if (!(eps >= 0.0f)) return set_error(PC_ERR_ARGUMENT, "eps must be non-negative");
  if (!aligned(values, 16) || !aligned(scales, 4) || !aligned(hidden_out, 16) || !aligned(hidden, 16) ||
      !aligned(delta, 16) || !aligned(parts, 16) || !aligned(weight, 16)) {
    return set_error(PC_ERR_ARGUMENT, "buffers must be 16-byte aligned, scales 4-byte aligned");
  }
  (void)hipGetLastError();
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows)), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const _Float16*>(hidden), parts ? static_cast<const void*>(parts) : delta, rows * width,
                       static_cast<const _Float16*>(weight), static_cast<_Float16*>(hidden_out), static_cast<uint8_t*>(values),
                       splits, width, static_cast<uint8_t*>(scales), eps);
  };
  auto with_delta = [&](auto instance) {
    constexpr int D = decltype(instance)::value;
    const bool full = width % (8 * kThreads) == 0;
    switch ((width / 8 - 1) / kThreads) {
      case 0: return full ? launch(add_rms_norm_fp8_kernel<1, true, D>) : launch(add_rms_norm_fp8_kernel<1, false, D>);
      case 1: return launch(add_rms_norm_fp8_kernel<2, false, D>);
      case 2: return launch(add_rms_norm_fp8_kernel<3, false, D>);
      default: return launch(add_rms_norm_fp8_kernel<4, false, D>);
    }
  };
  // Two, four or eight parts at once where a thread has one chunk of them (the registers of more do not repay).
  const bool one_chunk = width <= 8 * kThreads;
  if (!parts && !delta) with_delta(std::integral_constant<int, kNoDelta>{});
  else if (delta) with_delta(std::integral_constant<int, kHalfDelta>{});
  else if (splits == 1) with_delta(std::integral_constant<int, 1>{});
  else if (splits == 2) with_delta(std::integral_constant<int, 2>{});
  else if (splits == 4 && one_chunk) with_delta(std::integral_constant<int, 4>{});
  else if (splits == 8 && one_chunk) with_delta(std::integral_constant<int, 8>{});
  else with_delta(std::integral_constant<int, kAnySplits>{});
  return check_launch("add_rms_norm_fp8");
}

}  // namespace

extern "C" {

int32_t pc_fp8_scale_stride(int32_t width) { return width < 1 || width > kMaxWidth ? 0 : scale_stride(width); }

int pc_quantize_fp8(void* values, void* scales, const void* x, int64_t x_stride, int64_t rows, int32_t width, void* stream) {
  if (rows < 0) return set_error(PC_ERR_ARGUMENT, "negative row count");
  if (width < 16 || width % 16 != 0 || width > kMaxWidth) {
    return set_error(PC_ERR_ARGUMENT, "width %d must be a multiple of 16 in [16, %d]", width, kMaxWidth);
  }
  if (rows == 0) return ok();  // nothing to read or write (empty buffers may be null)
  if (!values || !scales || !x) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (x_stride < width || x_stride % 8 != 0) {
    return set_error(PC_ERR_ARGUMENT, "x_stride %lld must be >= %d and a multiple of 8", static_cast<long long>(x_stride), width);
  }
  if (!aligned(values, 16) || !aligned(scales, 4) || !aligned(x, 16)) {
    return set_error(PC_ERR_ARGUMENT, "values and x must be 16-byte aligned, scales 4-byte aligned");
  }
  const int32_t row_blocks = (width + kBlock - 1) / kBlock;
  constexpr int kPerGroup = kTurns * kThreads / 16;
  if (rows > (kMaxQuantizeBlocks - kPerGroup) / row_blocks) return set_error(PC_ERR_ARGUMENT, "quantize_fp8 too large");
  const uint32_t blocks = static_cast<uint32_t>(rows * row_blocks);
  (void)hipGetLastError();
  hipLaunchKernelGGL(quantize_fp8_kernel, dim3((blocks + kPerGroup - 1) / kPerGroup), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales),
                     static_cast<const _Float16*>(x), x_stride, blocks, static_cast<uint32_t>(row_blocks), width);
  return check_launch("quantize_fp8");
}

int pc_add_rms_norm_fp8(void* values, void* scales, void* hidden_out, const void* hidden, const void* delta,
                        const void* weight, int64_t rows, int32_t width, float eps, void* stream) {
  return add_rms_norm_fp8(values, scales, hidden_out, hidden, delta, nullptr, 1, weight, rows, width, eps, stream);
}

int pc_add_rms_norm_parts_fp8(void* values, void* scales, void* hidden_out, const void* hidden, const float* delta_parts,
                              int32_t splits, const void* weight, int64_t rows, int32_t width, float eps, void* stream) {
  if (rows > 0 && !delta_parts) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (splits < 1 || splits > 64) return set_error(PC_ERR_ARGUMENT, "splits %d outside [1, 64]", splits);
  return add_rms_norm_fp8(values, scales, hidden_out, hidden, nullptr, delta_parts, splits, weight, rows, width, eps, stream);
}

}  // extern "C"
