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

// One block of 128 columns per 16 lanes. What bounds it: HBM (2 bytes read, 1 written per element).
__global__ __launch_bounds__(kThreads) void quantize_fp8_kernel(uint8_t* values, uint8_t* scales, const _Float16* x,
                                                                int64_t x_stride, int64_t blocks, int32_t row_blocks,
                                                                int32_t width) {
  const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + threadIdx.x / 16;
  if (block >= blocks) return;
  const int64_t row = block / row_blocks;
  const int in_row = static_cast<int>(block - row * row_blocks);
  const int column = in_row * kBlock + 8 * (threadIdx.x % 16);
  float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (column < width) {
    const half8_t v = *reinterpret_cast<const half8_t*>(x + row * x_stride + column);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = static_cast<float>(v[i]);
  }
  int scale;
  const uint2_t packed = round8(y, scale);
  if (column < width) *reinterpret_cast<uint2_t*>(values + row * width + column) = packed;
  if (threadIdx.x % 16 == 0) scales[row * scale_stride(width) + in_row] = static_cast<uint8_t>(scale);
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

constexpr int kNoDelta = -1, kHalfDelta = 0;  // else: that many fp32 partial sums (kAnySplits: `splits`)
constexpr int kAnySplits = 64;

// One workgroup per row, eight columns per thread and chunk. The sum of the residual stream is an
// fp16 row (the next layer's residual), rounded as the fp16 form rounds it; the mean of squares and the
// norm are fp32. What bounds it: at decode sizes one round trip of memory (every load is issued
// before the first wait), at prompt sizes HBM.
template <int CHUNKS, int DELTA>
__global__ __launch_bounds__(kThreads) void add_rms_norm_fp8_kernel(const _Float16* hidden, const void* delta,
                                                                    int64_t parts_stride, const _Float16* weight,
                                                                    _Float16* hidden_out, uint8_t* values, uint8_t* scales,
                                                                    int32_t splits, int32_t width, float eps) {
  __shared__ float wave_sums[kThreads / 64];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * width;
  const int tid = threadIdx.x;
  auto column = [&](int c) { return 8 * (tid + c * kThreads); };
  float h[CHUNKS][8];
  half8_t wt[CHUNKS];
  float squares = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[c][i] = 0.0f;
    if (column(c) >= width) continue;
    const int64_t at = base + column(c);
    half8_t sum = *reinterpret_cast<const half8_t*>(hidden + at);
    wt[c] = *reinterpret_cast<const half8_t*>(weight + column(c));
    if constexpr (DELTA != kNoDelta) {
      half8_t d;
      if constexpr (DELTA == kHalfDelta) {
        d = *reinterpret_cast<const half8_t*>(static_cast<const _Float16*>(delta) + at);
      } else {
        const float* parts = static_cast<const float*>(delta) + at;
        float4_t lo = *reinterpret_cast<const float4_t*>(parts), hi = *reinterpret_cast<const float4_t*>(parts + 4);
        for (int s = 1; s < (DELTA == kAnySplits ? splits : DELTA); ++s) {
          lo += *reinterpret_cast<const float4_t*>(parts + s * parts_stride);
          hi += *reinterpret_cast<const float4_t*>(parts + s * parts_stride + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[i] = static_cast<_Float16>(lo[i]);
          d[i + 4] = static_cast<_Float16>(hi[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = static_cast<_Float16>(static_cast<float>(sum[i]) + static_cast<float>(d[i]));
    }
    if (hidden_out != nullptr) *reinterpret_cast<half8_t*>(hidden_out + at) = sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[c][i] = static_cast<float>(sum[i]);
      squares += h[c][i] * h[c][i];
    }
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
    const bool mine = column(c) < width;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = mine ? h[c][i] * static_cast<float>(wt[c][i]) * norm : 0.0f;  // the first product is exact
    int scale;
    const uint2_t packed = round8(y, scale);
    if (!mine) continue;
    *reinterpret_cast<uint2_t*>(values + base + column(c)) = packed;
    if (tid % 16 == 0) {
      scales[static_cast<int64_t>(blockIdx.x) * scale_stride(width) + column(c) / kBlock] = static_cast<uint8_t>(scale);
    }
  }
}

int add_rms_norm_fp8(void* values, void* scales, void* hidden_out, const void* hidden, const void* delta,
                     const float* parts, int32_t splits, const void* weight, int64_t rows, int32_t width, float eps,
                     void* stream) {
  if (rows < 0 || rows > INT32_MAX) return set_error(PC_ERR_ARGUMENT, "rows %lld out of range", static_cast<long long>(rows));
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
                       static_cast<const _Float16*>(weight), static_cast<_Float16*>(hidden_out),
                       static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales), splits, width, eps);
  };
  auto with_delta = [&](auto instance) {
    constexpr int D = decltype(instance)::value;
    switch ((width / 8 - 1) / kThreads) {
      case 0: return launch(add_rms_norm_fp8_kernel<1, D>);
      case 1: return launch(add_rms_norm_fp8_kernel<2, D>);
      case 2: return launch(add_rms_norm_fp8_kernel<3, D>);
      default: return launch(add_rms_norm_fp8_kernel<4, D>);
    }
  };
  if (parts) with_delta(std::integral_constant<int, kAnySplits>{});
  else if (delta) with_delta(std::integral_constant<int, kHalfDelta>{});
  else with_delta(std::integral_constant<int, kNoDelta>{});
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
  if (rows > (int64_t{INT32_MAX} * (kThreads / 16)) / row_blocks) return set_error(PC_ERR_ARGUMENT, "quantize_fp8 too large");
  const int64_t blocks = rows * row_blocks;
  (void)hipGetLastError();
  hipLaunchKernelGGL(quantize_fp8_kernel, dim3(static_cast<uint32_t>((blocks + kThreads / 16 - 1) / (kThreads / 16))),
                     dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<uint8_t*>(values),
                     static_cast<uint8_t*>(scales), static_cast<const _Float16*>(x), x_stride, blocks, row_blocks, width);
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
