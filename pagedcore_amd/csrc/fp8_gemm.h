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
  kRope,  // pc_qkv_rope_append_fp8
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

int launch_stream(const Args& a, Form form, hipStream_t s);  // not kSwiGLUFp8
int launch_tiles(const Args& a, Form form, hipStream_t s);   // not kPartials, e4m3 x

}  // namespace fp8_gemm

#endif  // PAGEDCORE_FP8_GEMM_H
