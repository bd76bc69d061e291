// Entry points of the 8-bit projections: the checks of their arguments, and which kernel takes a call.

#include "fp8_gemm.h"

namespace {

using namespace fp8_gemm;
using pc_internal::aligned;
using pc_internal::set_error;

constexpr int kMaxRows = 1 << 16;
constexpr int kMaxK = 1 << 22;     // tile-relative byte offsets fit 32 bits
constexpr int kMaxQkvK = 1 << 18;  // 2560 rows of W within 32-bit offsets
constexpr int kStreamRows = PC_FP8_STREAM_ROWS;  // of fp16 x and of fp32 partial sums

// The checks of what both entry points read; PC_OK, or an error.
int check_operands(const Args& a) {
  if (!a.x || !a.w || !a.w_scales) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.x_scales, 4) || !aligned(a.w_scales, 4)) {
    return set_error(PC_ERR_ARGUMENT, "x and w must be 16-byte aligned, scales 4-byte aligned");
  }
  return PC_OK;
}

// The checks of the sizes.
int check_sizes(const Args& a, Form form, bool half_x) {
  const int max_k = form == kRope ? kMaxQkvK : kMaxK;
  if (a.n < 1) return set_error(PC_ERR_ARGUMENT, "n must be positive");
  if (a.m < 1 || a.m > kMaxRows) return set_error(PC_ERR_ARGUMENT, "m = %d outside [1, %d]", a.m, kMaxRows);
  if (a.k < 16 || a.k % 16 != 0 || a.k > max_k) {
    return set_error(PC_ERR_ARGUMENT, "k = %d must be a multiple of 16 in [16, %d]", a.k, max_k);
  }
  if (static_cast<int64_t>(a.m) * a.k > (int64_t{1} << 31) || static_cast<int64_t>(a.n) * a.k > (int64_t{1} << 31)) {
    return set_error(PC_ERR_ARGUMENT, "GEMM of %d x %d x %d too large", a.m, a.n, a.k);
  }
  if (half_x && a.m > kStreamRows) {
    return set_error(PC_ERR_ARGUMENT, "fp16 x takes up to %d rows: quantize %d rows first", kStreamRows, a.m);
  }
  const int columns = form == kSwiGLUFp8 ? 32 : form == kSwiGLU ? 8 : 4;
  if (a.n % columns != 0) return set_error(PC_ERR_ARGUMENT, "n = %d must be a multiple of %d", a.n, columns);
  if (form == kPartials) {
    const int blocks = (a.k + PC_FP8_BLOCK - 1) / PC_FP8_BLOCK;
    if (a.splits < 1 || a.splits > 64 || a.splits > blocks) {
      return set_error(PC_ERR_ARGUMENT, "splits %d outside [1, 64] or more than k's %d blocks", a.splits, blocks);
    }
    if (a.m > kStreamRows) return set_error(PC_ERR_ARGUMENT, "fp32 partial sums take up to %d rows, not %d", kStreamRows, a.m);
  } else if (a.splits != 1) {
    return set_error(PC_ERR_ARGUMENT, "only partial sums take splits");
  }
  if (static_cast<int64_t>(a.splits) * a.m * a.n > (int64_t{1} << 31)) {  // keeps a grid's threads within 32 bits, too
    return set_error(PC_ERR_ARGUMENT, "GEMM of %d x %d x %d with %d splits too large", a.m, a.n, a.k, a.splits);
  }
  if (form == kSwiGLUFp8 && half_x) return set_error(PC_ERR_ARGUMENT, "PC_GEMM_SWIGLU_FP8 takes 8-bit x");
  return PC_OK;
}

bool known(int32_t epilogue) {
  return epilogue == PC_GEMM_PARTIALS || epilogue == PC_GEMM_HALF || epilogue == PC_GEMM_SWIGLU || epilogue == PC_GEMM_SWIGLU_FP8;
}

// fp32 partial sums and fp16 x are the streams' alone, 8-bit outputs the tiles'.
bool streams(Form form) { return form != kSwiGLUFp8; }
bool tiles(Form form, bool half_x) { return form != kPartials && !half_x; }

// The kernel with the shorter estimate: an index among the form's streams, and its tiles behind them.
int choose(const Args& a, Form form, bool half_x) {
  const Choice stream = streams(form) ? choose_stream(a, form, half_x) : Choice{-1, INFINITY};
  const Choice tile = tiles(form, half_x) ? choose_tile(a, form) : Choice{-1, INFINITY};
  return stream.time <= tile.time ? stream.index : (streams(form) ? stream_kernels(form, half_x) : 0) + tile.index;
}

int launch(const Args& a, Form form, hipStream_t s) {
  (void)hipGetLastError();
  const bool half_x = !a.x_scales;
  const int index = choose(a, form, half_x), first_tile = streams(form) ? stream_kernels(form, half_x) : 0;
  return index < first_tile ? launch_stream(a, form, index, s) : launch_tile(a, form, index - first_tile, s);
}

}  // namespace

extern "C" {

int pc_gemm_fp8(void* out, void* out_scales, const void* x, const void* x_scales, const void* w, const void* w_scales,
                int32_t m, int32_t n, int32_t k, int32_t splits, int32_t epilogue, void* stream) {
  Args a{};
  a.x = x;
  a.x_scales = static_cast<const uint8_t*>(x_scales);
  a.w = static_cast<const uint8_t*>(w);
  a.w_scales = static_cast<const uint8_t*>(w_scales);
  a.m = m;
  a.n = n;
  a.k = k;
  a.splits = splits;
  a.out = out;
  a.out_scales = static_cast<uint8_t*>(out_scales);
  if (!out) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (int rc = check_operands(a)) return rc;
  if (!aligned(out, 16) || !aligned(out_scales, 4)) {
    return set_error(PC_ERR_ARGUMENT, "out must be 16-byte aligned, scales 4-byte aligned");
  }
  if (!known(epilogue)) return set_error(PC_ERR_ARGUMENT, "unknown epilogue %d", epilogue);
  const Form form = static_cast<Form>(epilogue);
  if ((out_scales != nullptr) != (form == kSwiGLUFp8)) {
    return set_error(PC_ERR_ARGUMENT, "out_scales belong to PC_GEMM_SWIGLU_FP8, and only to it");
  }
  if (int rc = check_sizes(a, form, !x_scales)) return rc;
  return launch(a, form, static_cast<hipStream_t>(stream));
}

int32_t pc_gemm_fp8_kernels(int32_t epilogue, int32_t half_x) {
  if (!known(epilogue) && epilogue != PC_GEMM_QKV_ROPE) return 0;
  const Form form = static_cast<Form>(epilogue);
  if (half_x && !streams(form)) return 0;
  return (streams(form) ? stream_kernels(form, half_x) : 0) + (tiles(form, half_x) ? tile_kernels(form) : 0);
}

int32_t pc_gemm_fp8_kernel(int32_t m, int32_t n, int32_t k, int32_t splits, int32_t epilogue, int32_t half_x) {
  Args a{};
  a.m = m;
  a.n = n;
  a.k = k;
  a.splits = splits;
  if (!known(epilogue) && epilogue != PC_GEMM_QKV_ROPE) return -1;
  const Form form = static_cast<Form>(epilogue);
  if (check_sizes(a, form, half_x) != PC_OK || (form == kRope && n != rope_device::kQkvElems)) return -1;
  return choose(a, form, half_x);
}

int pc_qkv_rope_append_fp8(void* query_out, void* key_out, void* value_out, const void* x, const void* x_scales,
                           const void* w, const void* w_scales, int32_t m, int32_t k, const int64_t* positions,
                           const void* rope_table, int32_t rope_positions, void* pool, int64_t num_blocks, int32_t layer,
                           const int64_t* slot_mapping, void* stream) {
  using namespace rope_device;
  Args a{};
  a.x = x;
  a.x_scales = static_cast<const uint8_t*>(x_scales);
  a.w = static_cast<const uint8_t*>(w);
  a.w_scales = static_cast<const uint8_t*>(w_scales);
  a.m = m;
  a.n = kQkvElems;
  a.k = k;
  a.splits = 1;
  if (!query_out || !positions || !rope_table) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (int rc = check_operands(a)) return rc;
  if (int rc = check_sizes(a, kRope, !x_scales)) return rc;
  if (rope_positions < 1) return set_error(PC_ERR_ARGUMENT, "rope_positions must be positive");
  if ((pool == nullptr) != (slot_mapping == nullptr)) {
    return set_error(PC_ERR_ARGUMENT, "pool and slot_mapping must both be given or both be null");
  }
  if (pool != nullptr) {
    if (num_blocks < 1 || num_blocks > INT32_MAX) {
      return set_error(PC_ERR_ARGUMENT, "num_blocks %lld out of range", static_cast<long long>(num_blocks));
    }
    if (layer < 0 || layer >= kLayers) return set_error(PC_ERR_ARGUMENT, "layer %d outside [0, 22)", layer);
  }
  if (!aligned(query_out, 16) || !aligned(key_out, 16) || !aligned(value_out, 16) || !aligned(rope_table, 16) || !aligned(pool, 16)) {
    return set_error(PC_ERR_ARGUMENT, "buffers must be 16-byte aligned");
  }
  a.positions = positions;
  a.slots = slot_mapping;
  a.rope.table = static_cast<const _Float16*>(rope_table);
  a.rope.table_positions = rope_positions;
  a.rope.query = static_cast<_Float16*>(query_out);
  a.rope.kind_elems = pool ? num_blocks * kSlots * kRowElems : 0;
  a.rope.layer_pool = pool ? static_cast<_Float16*>(pool) + static_cast<int64_t>(layer) * 2 * a.rope.kind_elems : nullptr;
  a.rope.key = static_cast<_Float16*>(key_out);
  a.rope.value = static_cast<_Float16*>(value_out);
  return launch(a, kRope, static_cast<hipStream_t>(stream));
}

}  // extern "C"
