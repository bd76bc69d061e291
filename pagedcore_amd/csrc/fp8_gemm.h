// What the kernels of the 8-bit projections and their entry points share (not part of the C ABI).
#ifndef PAGEDCORE_FP8_GEMM_H
#define PAGEDCORE_FP8_GEMM_H

#include <stdint.h>

#include <hip/hip_runtime.h>

#include "fp8_device.h"
#include "gemm_device.h"

namespace fp8_gemm {

enum Form : int32_t {
  kPartials = PC_GEMM_PARTIALS,
  kHalf = PC_GEMM_HALF,
  kSwiGLU = PC_GEMM_SWIGLU,
  kSwiGLUFp8 = PC_GEMM_SWIGLU_FP8,
  kRope = PC_GEMM_QKV_ROPE,
};
// The forms whose tiles hold pairs of W rows: gate and up, or a head's d and d + 32.
constexpr bool paired(Form f) { return f == kSwiGLU || f == kSwiGLUFp8 || f == kRope; }

struct Args {
  const void* x;            // e4m3 [m][k], or fp16 (x_scales null)
  const uint8_t* x_scales;  // [m][scale_stride(k)]
  const uint8_t* w;         // e4m3 [n][k]
  const uint8_t* w_scales;  // [n][scale_stride(k)]
  int m, n, k, splits;
  void* out;
  uint8_t* out_scales;       // kSwiGLUFp8
  const int64_t* positions;  // kRope, and the rest
  const int64_t* slots;
  rope_device::RopeOut rope;
};

// A kernel instance that can take a call, and the estimate of its time (us).
struct Choice {
  int index;
  float time;
};

// An estimate's constants: a launch, a round of workgroups on the CUs, a block of 128 columns of one round (the
// slowest wave's), 10^6 bytes of weight.
struct Cost {
  float launch, round, block, weight;
};
inline float estimate(const Cost& c, int64_t workgroups, int blocks, const Args& a) {
  const float rounds = static_cast<float>((workgroups + 255) / 256);
  return c.launch + rounds * (c.round + c.block * blocks) + c.weight * 1e-6f * static_cast<float>(a.n) * static_cast<float>(a.k);
}

// A q|k|v product, as fp16 or rotated: both take the same instance, so that they have the same bits.
inline bool qkv_product(const Args& a, Form form) { return form == kRope || (form == kHalf && a.n == rope_device::kQkvElems); }

// Of the sizes in `a` and of whether x is fp16, and of nothing else in it.
Choice choose_stream(const Args& a, Form form, bool half_x);  // not kSwiGLUFp8
Choice choose_tile(const Args& a, Form form);                 // not kPartials, e4m3 x
int stream_kernels(Form form, bool half_x);                   // how many each chooses among
int tile_kernels(Form form);
int launch_stream(const Args& a, Form form, int index, hipStream_t s);
int launch_tile(const Args& a, Form form, int index, hipStream_t s);

}  // namespace fp8_gemm

#endif  // PAGEDCORE_FP8_GEMM_H
