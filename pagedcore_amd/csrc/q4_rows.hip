// Rows of the 4-bit KV pool: quantised as they are written (pc_kv_append_q4), and read back as fp16
// (pc_kv_read_q4). The format and its bytes are in q4_device.h. Both are bound by HBM: 1024 bytes of fp16 and
// 288 of the pool per token and layer.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "pagedcore_hip.h"
#include "pc_internal.h"
#include "q4_device.h"

namespace {

using namespace q4_device;
using pc_internal::aligned;
using pc_internal::check_launch;
using pc_internal::ok;
using pc_internal::set_error;

constexpr int kThreads = 256;
constexpr int kRowsPerGroup = kThreads / kRowLanes;

struct RowArgs {
  char* key;  // fp16 rows; strides in bytes
  char* value;
  int64_t key_layer, key_token, value_layer, value_token;
  const int64_t* slots;
  char* pool;
  int64_t num_blocks;
  uint32_t tokens, rows;  // rows = layers * tokens * 2 kinds * 4 heads
  int32_t layer_begin;
};

struct Row {
  char* half;  // the fp16 row
  char* unit;  // null: its slot lies outside the pool
  int kind, t;
};

__device__ __forceinline__ Row row_of(const RowArgs& args, uint32_t row) {
  const uint32_t h = row % kKVHeads, kind = row / kKVHeads % 2, rest = row / (2 * kKVHeads);
  const uint32_t token = rest % args.tokens, layer = rest / args.tokens;
  const int64_t slot = args.slots[token];
  Row r;
  r.half = (kind ? args.value + layer * args.value_layer + token * args.value_token
                 : args.key + layer * args.key_layer + token * args.key_token) + h * (2 * kHeadDim);
  r.kind = static_cast<int>(kind);
  r.t = static_cast<int>(slot & (kSlots - 1));
  const bool inside = slot >= 0 && slot < args.num_blocks * kSlots;
  r.unit = inside ? args.pool + ((static_cast<int64_t>(args.layer_begin + layer) * args.num_blocks + slot / kSlots) * kKVHeads + h) * kUnitBytes
                  : nullptr;
  return r;
}

// VEC: the rows are 16-byte aligned; else they are read and written a value at a time.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void kv_append_q4_kernel(RowArgs args) {
  const uint32_t row = blockIdx.x * kRowsPerGroup + threadIdx.x / kRowLanes;
  if (row >= args.rows) return;
  const int a = threadIdx.x % kRowLanes;
  const Row r = row_of(args, row);
  half8_t x;
  if constexpr (VEC) {
    x = *reinterpret_cast<const half8_t*>(r.half + 16 * a);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = reinterpret_cast<const _Float16*>(r.half)[8 * a + j];
  }
  const Levels q = quantize8(x);
  if (r.unit != nullptr) store_row(r.unit, r.kind, r.t, a, q);
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void kv_read_q4_kernel(RowArgs args) {
  const uint32_t row = blockIdx.x * kRowsPerGroup + threadIdx.x / kRowLanes;
  if (row >= args.rows) return;
  const int a = threadIdx.x % kRowLanes;
  const Row r = row_of(args, row);
  if (r.unit == nullptr) return;
  const uint32_t pair = *reinterpret_cast<const uint32_t*>(r.unit + pair_offset(r.kind, r.t));
  uint32_t n[8];
  if (r.kind == 0) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(r.unit + key_word(r.t, a));
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = level(word, j);
  } else {
    const char* at = r.unit + value_byte(r.t, a);
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = static_cast<uint8_t>(at[16 * j]) >> (a & 2 ? 4 : 0) & 15u;
  }
  const half8_t x = row_values(pair, n);
  if constexpr (VEC) {
    *reinterpret_cast<half8_t*>(r.half + 16 * a) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) reinterpret_cast<_Float16*>(r.half)[8 * a + j] = x[j];
  }
}

// Checks of both entry points; PC_OK with args filled in, or an error.
int row_args(RowArgs& args, const void* pool, int64_t num_blocks, int32_t layer_begin, int32_t num_layers, const void* key,
             int64_t key_layer_stride, int64_t key_token_stride, const void* value, int64_t value_layer_stride,
             int64_t value_token_stride, const int64_t* slot_mapping, int64_t num_tokens) {
  if (!pool || !key || !value || !slot_mapping) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (num_blocks < 1 || num_blocks > (1 << 26)) return set_error(PC_ERR_ARGUMENT, "num_blocks %lld out of range [1, 2^26]", static_cast<long long>(num_blocks));
  if (num_layers < 1 || layer_begin < 0 || num_layers > kLayers || layer_begin > kLayers - num_layers) {
    return set_error(PC_ERR_ARGUMENT, "layers [%d, %d + %d) outside [0, %d)", layer_begin, layer_begin, num_layers, kLayers);
  }
  if (num_tokens < 0) return set_error(PC_ERR_ARGUMENT, "negative token count");
  if (num_tokens > (int64_t{1} << 31) / (num_layers * 2 * kKVHeads)) {
    return set_error(PC_ERR_ARGUMENT, "%lld tokens of %d layers are too many", static_cast<long long>(num_tokens), num_layers);
  }
  if (!aligned(pool, 128)) return set_error(PC_ERR_ARGUMENT, "pool must be 128-byte aligned");
  if (!aligned(key, 2) || !aligned(value, 2)) return set_error(PC_ERR_ARGUMENT, "K/V must be 2-byte aligned");
  if (!aligned(slot_mapping, 8)) return set_error(PC_ERR_ARGUMENT, "slot_mapping must be 8-byte aligned");
  args.key = const_cast<char*>(static_cast<const char*>(key));
  args.value = const_cast<char*>(static_cast<const char*>(value));
  args.key_layer = key_layer_stride * 2;
  args.key_token = key_token_stride * 2;
  args.value_layer = value_layer_stride * 2;
  args.value_token = value_token_stride * 2;
  args.slots = slot_mapping;
  args.pool = const_cast<char*>(static_cast<const char*>(pool));
  args.num_blocks = num_blocks;
  args.tokens = static_cast<uint32_t>(num_tokens);
  args.rows = static_cast<uint32_t>(num_tokens * num_layers * 2 * kKVHeads);
  args.layer_begin = layer_begin;
  return PC_OK;
}

bool rows_aligned(const RowArgs& args) {
  return aligned(args.key, 16) && aligned(args.value, 16) && args.key_layer % 16 == 0 && args.key_token % 16 == 0 &&
         args.value_layer % 16 == 0 && args.value_token % 16 == 0;
}

unsigned grid_of(const RowArgs& args) { return (args.rows + kRowsPerGroup - 1) / kRowsPerGroup; }

}  // namespace

extern "C" {

int pc_kv_append_q4(void* pool, int64_t num_blocks, int32_t layer_begin, int32_t num_layers, const void* key,
                    int64_t key_layer_stride, int64_t key_token_stride, const void* value, int64_t value_layer_stride,
                    int64_t value_token_stride, const int64_t* slot_mapping, int64_t num_tokens, void* stream) {
  RowArgs args;
  if (int rc = row_args(args, pool, num_blocks, layer_begin, num_layers, key, key_layer_stride, key_token_stride, value,
                        value_layer_stride, value_token_stride, slot_mapping, num_tokens)) {
    return rc;
  }
  if (args.rows == 0) return ok();
  (void)hipGetLastError();
  hipLaunchKernelGGL(rows_aligned(args) ? kv_append_q4_kernel<true> : kv_append_q4_kernel<false>, dim3(grid_of(args)), dim3(kThreads),
                     0, static_cast<hipStream_t>(stream), args);
  return check_launch("kv_append_q4");
}

int pc_kv_read_q4(void* key, int64_t key_layer_stride, int64_t key_token_stride, void* value, int64_t value_layer_stride,
                  int64_t value_token_stride, const void* pool, int64_t num_blocks, int32_t layer_begin, int32_t num_layers,
                  const int64_t* slot_mapping, int64_t num_tokens, void* stream) {
  RowArgs args;
  if (int rc = row_args(args, pool, num_blocks, layer_begin, num_layers, key, key_layer_stride, key_token_stride, value,
                        value_layer_stride, value_token_stride, slot_mapping, num_tokens)) {
    return rc;
  }
  if (args.rows == 0) return ok();
  (void)hipGetLastError();
  hipLaunchKernelGGL(rows_aligned(args) ? kv_read_q4_kernel<true> : kv_read_q4_kernel<false>, dim3(grid_of(args)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), args);
  return check_launch("kv_read_q4");
}

}  // extern "C"
