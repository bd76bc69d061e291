// Device helpers of the 8-bit rows, shared by the kernels that write and read them (not part of the
// C ABI): e4m3 values with one power of two per row and block of 128 columns.
//
// The scale of a block is the smallest power of two with which its largest magnitude does not pass
// 448, e4m3's largest value. A power of two, because e4m3's relative step is the same at every power
// (a free scale would gain nothing but part of a binade at the subnormal end, 15 binades down), because
// scaling by it is exact, and because the scaled matrix instruction takes it as it is stored.
#ifndef PAGEDCORE_FP8_DEVICE_H
#define PAGEDCORE_FP8_DEVICE_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "pagedcore_hip.h"

namespace fp8_device {

constexpr int kBlock = PC_FP8_BLOCK;  // columns that share a scale

// Bytes between the scales of two rows: a row's scales are read four at a time.
__host__ __device__ constexpr int scale_stride(int k) { return (k + 4 * kBlock - 1) / (4 * kBlock) * 4; }

// The biased exponent of the scale of a block whose largest magnitude is `largest` (finite, >= 0):
// with largest = f 2^e, f in [1, 2), 448 = 1.75 2^8 is not passed at e - 8 if f <= 1.75, else at e - 7.
// Adding 0x1fffff to the bits carries into the exponent where the fraction is above 0.75.
__device__ __forceinline__ int scale_of(float largest) {
  return max(1, static_cast<int>((__float_as_uint(largest) + 0x1fffffu) >> 23) - 8);
}
// 2^(s - 127) and 2^(127 - s), s in [1, 253].
__device__ __forceinline__ float power_of(int s) { return __uint_as_float(static_cast<uint32_t>(s) << 23); }
__device__ __forceinline__ float inverse_of(int s) { return __uint_as_float(static_cast<uint32_t>(254 - s) << 23); }

// Four values, already divided by their scale, rounded to e4m3 (to nearest even; infinities and NaN
// become NaN).
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return static_cast<uint32_t>(v);
}

// silu(gate) * up in fp32, silu(x) = x / (1 + e^-x), with the hardware's base-2 exponential and reciprocal (one
// ulp each; the exponent's own rounding adds |x| 2^-24). The outputs are rounded to fp16 or to 8 bits; expf and
// a correctly rounded quotient are several times the instructions beside the tiles' products (without them, and with the
// next stage read before the refill, SwiGLU of 2048 rows 63.4 -> 56.6 us).
__device__ __forceinline__ float silu_mul(float gate, float up) {
  const float e = __builtin_amdgcn_exp2f(gate * -1.44269504088896340736f);
  return gate * __builtin_amdgcn_rcpf(1.0f + e) * up;
}

// |x| if it is finite, else 0: an infinity or NaN becomes a NaN of its own and leaves the scale, and
// with it the block's other values, alone.
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

template <int CTRL>
__device__ __forceinline__ float max_dpp(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false)));
}
// The largest over the 16 lanes of a row of the wave, in each of them (rotations by 8, 4, 2 and 1).
__device__ __forceinline__ float max16(float x) {
  x = max_dpp<0x128>(x);
  x = max_dpp<0x124>(x);
  x = max_dpp<0x122>(x);
  return max_dpp<0x121>(x);
}

}  // namespace fp8_device

#endif  // PAGEDCORE_FP8_DEVICE_H
