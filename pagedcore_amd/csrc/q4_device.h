// Device helpers of the 4-bit KV pool, shared by the kernels that write and read it (not part of the
// C ABI): a row's quantisation and where its bytes lie.
//
// A row (64 values of one token, kv head and kind) is held as lo = min(x), s = the smallest fp16 with
// 15 s >= max(x) - lo and the levels n = round_half_even((x - lo) / s), for the values lo + s n. s is
// rounded up, so no level passes 15 and none needs a clamp; lo is one of the values, so it needs no rounding. The two
// differences are fp32's: exact but in rows whose magnitudes span more than 2^13.
// Scale and minimum belong to a row, not to a channel: they then leave the attention's products, which
// multiply the levels alone (s and lo enter once per token, in fp32).
//
// A unit (one block of 16 tokens, one kv head) is 1152 bytes, nine 128-byte lines: K's levels (512 bytes), V's
// (512), then (lo, s) as fp16 pairs of the 16 K rows (64) and of the 16 V rows (64). Within them the levels lie as
// the matrix instruction's lanes take them, 16 bytes a lane, and every token has bytes of its own, so that rows are
// written without reading their neighbours:
//   K: token 4i + e (i, e in 0..3), dims 32 x + 8 g + j (x in 0..1, g in 0..3, j in 0..7): the word at
//      256 (i / 2) + 64 e + 16 g + 8 (i % 2) + 4 x, bits 4 (j / 2) + 16 (j % 2)
//   V: token 4q + t, dims 32 p + r (low half) and 32 p + 16 + r (high half of the byte, r in 0..15): the byte at
//      256 (q / 2) + 16 r + 8 (q % 2) + 4 p + {0, 2, 1, 3}[t]
// In both, a 16-bit half of (word >> 4 n) & 0x000F000F is one of two neighbours of the product's inner index.
#ifndef PAGEDCORE_Q4_DEVICE_H
#define PAGEDCORE_Q4_DEVICE_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "attn_plan.h"
#include "pc_device.h"
#include "pagedcore_hip.h"

namespace q4_device {

using attn_plan::kHeadDim;
using attn_plan::kKVHeads;
using attn_plan::kLayers;
using attn_plan::kSlots;
using pc_device::half8_t;

constexpr int kUnitBytes = PC_Q4_UNIT_BYTES;
constexpr int kValueOffset = 512;
constexpr int kPairOffset = 1024;       // (lo, s) of the K rows; the V rows' follow
constexpr int kPairBytes = 4 * kSlots;  // 64
constexpr int64_t kBlockBytes = kKVHeads * kUnitBytes;
constexpr int kRowLanes = 8;  // lanes of a row, 8 values each
static_assert(kUnitBytes == kPairOffset + 2 * kPairBytes, "K, V, and the pairs of both");

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), CTRL, 0xf, 0xf, true));  // every lane has a source
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(x)));
}
constexpr int kSwap1 = 0xB1;     // quad_perm [1, 0, 3, 2]
constexpr int kSwap2 = 0x4E;     // quad_perm [2, 3, 0, 1]
constexpr int kMirror8 = 0x141;  // row_half_mirror: lane 7 - l of its eight
constexpr int kRotate8 = 0x128;  // row_ror 8: lane l ^ 8 of a row of 16

// One eighth of a quantised row: its 8 levels as the K word above, and the row's (lo, s) as the pair's bits.
struct Levels {
  uint32_t word;
  uint32_t pair;
};

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ half2_t dpp(half2_t x) {
  return __builtin_bit_cast(half2_t, dpp<CTRL>(__builtin_bit_cast(uint32_t, x)));
}

// Lane a of eight (aligned) holds values 8a .. 8a + 7 of a row. Its minimum and maximum are taken on pairs, by the forms that
// hand a NaN on. The quotient t / s ends correctly rounded: t s^-1 with a reciprocal good to an ulp, and one step with the
// exact residual (Markstein): what is left of the error is 2^-45 of it, and a quotient at a half (a tie, to the even level)
// or next to one is 2^-21 from any other value that 24 bits of t and 11 of s give. (lo, s) of a row with an infinity or NaN
// is (NaN, 0): all its values are NaN.
__device__ __forceinline__ Levels quantize8(half8_t x) {
#pragma clang fp contract(off)
  half2_t lo2 = {x[0], x[1]}, hi2 = lo2;
#pragma unroll
  for (int j = 2; j < 8; j += 2) {
    const half2_t v = {x[j], x[j + 1]};
    lo2 = __builtin_elementwise_minimum(lo2, v);
    hi2 = __builtin_elementwise_maximum(hi2, v);
  }
  lo2 = __builtin_elementwise_minimum(lo2, dpp<kSwap1>(lo2));
  hi2 = __builtin_elementwise_maximum(hi2, dpp<kSwap1>(hi2));
  lo2 = __builtin_elementwise_minimum(lo2, dpp<kSwap2>(lo2));
  hi2 = __builtin_elementwise_maximum(hi2, dpp<kSwap2>(hi2));
  lo2 = __builtin_elementwise_minimum(lo2, dpp<kMirror8>(lo2));
  hi2 = __builtin_elementwise_maximum(hi2, dpp<kMirror8>(hi2));
  // + 0: a zero of either sign is +0, the row's bytes do not depend on the order of its values.
  const float lo = static_cast<float>(__builtin_elementwise_minimum(lo2[0], lo2[1])) + 0.f;
  const float span = static_cast<float>(__builtin_elementwise_maximum(hi2[0], hi2[1])) - lo + 0.f;  // (-0 of a row of -0 alone)
  uint32_t step_bits = __builtin_bit_cast(uint16_t, static_cast<_Float16>(span * (1.0f / 15.0f)));
  // 15 s is exact in fp32 (4 and 11 bits).
  if (static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(step_bits))) * 15.0f < span) ++step_bits;
  const float step = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(step_bits)));
  const float inverse = step > 0.f ? __builtin_amdgcn_rcpf(step) : 0.f;
  // A one that the compiler does not see through: x 1 - lo is one instruction on the half, x - lo a conversion and a difference.
  float one;
  asm("s_mov_b32 %0, 1.0" : "=s"(one));
  uint32_t low = 0, high = 0;  // the levels of even and of odd j, in the low 16 bits
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = fmaf(static_cast<float>(x[j]), one, -lo);
    float y = t * inverse;
    y = fmaf(fmaf(-y, step, t), inverse, y);
    const uint32_t n = __float_as_uint(y + 8388608.0f);  // an integer, to nearest even, below bits 24 and on
    if (j % 2 == 0) low |= n << (2 * j);
    else high |= n << (2 * (j - 1));
  }
  Levels r;
  r.word = __builtin_amdgcn_perm(high, low, 0x05040100u);
  r.pair = __builtin_bit_cast(uint16_t, static_cast<_Float16>(lo)) | step_bits << 16;
  if (!(span < INFINITY)) {
    r.word = 0;
    r.pair = 0x7e00u;  // (NaN, 0)
  }
  return r;
}

// The level of value j of a lane's word.
__device__ __forceinline__ uint32_t level(uint32_t word, int j) { return word >> (4 * (j / 2) + 16 * (j % 2)) & 15u; }

// Offsets within a unit: lane a's K word of token t, the first of lane a's V bytes (dims r = 8 (a % 2) + j at + 16 j), and
// the row's pair.
__device__ __forceinline__ int key_word(int t, int a) {
  return 256 * (t >> 3) + 64 * (t & 3) + 16 * (a & 3) + 8 * (t >> 2 & 1) + 4 * (a >> 2);
}
__device__ __forceinline__ int value_byte(int t, int a) {
  const int place = (t & 1) << 1 | (t >> 1 & 1);  // 0, 2, 1, 3
  return kValueOffset + 256 * (t >> 3) + 128 * (a & 1) + 8 * (t >> 2 & 1) + 4 * (a >> 2) + place;
}
__device__ __forceinline__ int pair_offset(int kind, int t) { return kPairOffset + kPairBytes * kind + 4 * t; }

// Stores token t's row (lane a of eight, all of them here) into its unit. A V byte holds values of two lanes, a and
// a ^ 2: each stores the bytes of four of their eight columns.
__device__ __forceinline__ void store_row(char* unit, int kind, int t, int a, const Levels& q) {
  const uint32_t other = dpp<kSwap2>(q.word);
  if (kind == 0) {
    *reinterpret_cast<uint32_t*>(unit + key_word(t, a)) = q.word;
  } else {
    const bool upper = (a & 2) != 0;
    const uint32_t lo_word = upper ? other : q.word, hi_word = upper ? q.word : other;
    char* at = unit + value_byte(t, a) + (upper ? 64 : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n = upper ? level(lo_word, j + 4) | level(hi_word, j + 4) << 4 : level(lo_word, j) | level(hi_word, j) << 4;
      at[16 * j] = static_cast<char>(n);
    }
  }
  if (a == 0) *reinterpret_cast<uint32_t*>(unit + pair_offset(kind, t)) = q.pair;
}

__device__ __forceinline__ float pair_low(uint32_t pair) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(pair))); }
__device__ __forceinline__ float pair_step(uint32_t pair) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(pair >> 16))); }

// Eight values in fp16: the exact lo + s n, rounded to fp32 (it has at most 40 bits) and to fp16. s is rounded up, so lo + 15 s may
// pass 65504 where the row's largest value did not: it reads as 65504 (by a minimum that hands a NaN on, two values an instruction).
__device__ __forceinline__ half8_t row_values(float lo, float step, const float (&n)[8]) {
  half8_t x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = static_cast<_Float16>(fmaf(step, n[j], lo));
  const _Float16 most = static_cast<_Float16>(65504.f);
  return __builtin_elementwise_minimum(x, half8_t{most, most, most, most, most, most, most, most});
}

// Values 8a .. 8a + 7 of token t's row, lane a of eight.
__device__ __forceinline__ half8_t load_row(const char* unit, int kind, int t, int a) {
  const uint32_t pair = *reinterpret_cast<const uint32_t*>(unit + pair_offset(kind, t));
  uint32_t n[8];
  if (kind == 0) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(unit + key_word(t, a));
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = level(word, j);
  } else {
    const char* at = unit + value_byte(t, a);
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = static_cast<uint8_t>(at[16 * j]) >> (a & 2 ? 4 : 0) & 15u;
  }
  float levels[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) levels[j] = static_cast<float>(n[j]);
  return row_values(pair_low(pair), pair_step(pair), levels);
}

}  // namespace q4_device

#endif  // PAGEDCORE_Q4_DEVICE_H
