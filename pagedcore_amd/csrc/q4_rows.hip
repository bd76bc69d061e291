// Rows of the 4-bit KV pool: quantised as they are written (pc_kv_append_q4), and read back as fp16
// (pc_kv_read_q4). The format and its bytes are in q4_device.h. Both are bound by HBM, with vector instructions close behind
// (970 a wave of 64 rows in the append, 700 in the read, which took 12.7 us below and not 10.7 with 960): 1024 bytes of fp16 and
// 288 of the pool per token and layer. In a graph, with the launch, 2048 tokens of 22 layers (59 MB) are appended in 16.2 us and
// read back in 13.5 where every call has other data, 16384 in 88 and 81 (5.4 and 5.8 TB/s; a large fill reaches 6.9, a large
// copy 4.9). One call repeated finds its source in the last-level cache: 14.5 and 10.7, 88 and 69. The figures below are such.

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
  uint32_t begin;         // the launch's first row (eight lanes a row: a launch has less than 2^32 threads)
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
  const uint32_t row = args.begin + blockIdx.x * kRowsPerGroup + threadIdx.x / kRowLanes;
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
  const uint32_t row = args.begin + blockIdx.x * kRowsPerGroup + threadIdx.x / kRowLanes;
  if (row >= args.rows) return;
  const int a = threadIdx.x % kRowLanes;
  const Row r = row_of(args, row);
  if (r.unit == nullptr) return;
  const half8_t x = load_row(r.unit, r.kind, r.t, a);
  if constexpr (VEC) {
    *reinterpret_cast<half8_t*>(r.half + 16 * a) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) reinterpret_cast<_Float16*>(r.half)[8 * a + j] = x[j];
  }
}

// Eight tokens a wave, of all heads and both kinds: what a prompt's rows take. A wave of eight consecutive slots (from a multiple
// of eight on) turns its levels in registers into the unit's 16-byte chunks, so that it stores and loads whole chunks, 128
// bytes of eight lanes; other slots go a token at a time, as above.
constexpr int kGroupTokens = 8;
constexpr int kGroupWaves = 4;
// Rows (8 a token and layer) above which they pay: 1024 tokens of 1, 2 and 5 layers take 4.6, 4.6 and 4.8 us in groups, 3.2, 3.5 and 5.2
// a token at a time; 2048 of 22 layers 14.5 and 22.2, read back 10.7 and 21.5, 16384 read back 69 and 196.
constexpr uint32_t kGroupRows = 8 * 4400;

struct Group {
  int64_t slot;    // lane a of eight: of token a of the group, -1 if there is none or it lies outside the pool
  int64_t first;   // of token 0
  uint32_t layer;
  int64_t token0;  // may begin before token 0 and end behind the last
  bool whole;      // the eight slots are one half of a block
};

// Token groups begin where the first token's slot says that halves of blocks begin.
__device__ __forceinline__ bool group_of(const RowArgs& args, Group& g) {
  const uint32_t groups = (args.tokens + 2 * kGroupTokens - 2) / kGroupTokens;
  const uint32_t w = blockIdx.x * kGroupWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  g.layer = w / groups;
  if (g.layer >= args.rows / (args.tokens * 2 * kKVHeads)) return false;
  g.token0 = static_cast<int64_t>(w % groups) * kGroupTokens - (args.slots[0] & (kGroupTokens - 1));
  if (g.token0 >= args.tokens) return false;
  const int64_t token = g.token0 + threadIdx.x % kGroupTokens;
  const int64_t slot = args.slots[token < 0 ? 0 : token < args.tokens ? token : args.tokens - 1];
  g.slot = token >= 0 && token < args.tokens && slot >= 0 && slot < args.num_blocks * kSlots ? slot : -1;
  g.first = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(g.slot >> 32)))) << 32 |
                                 static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(g.slot))));
  const bool here = g.slot == g.first + threadIdx.x % kGroupTokens && g.first >= 0 && g.first % kGroupTokens == 0;
  g.whole = __builtin_amdgcn_ballot_w64(!here) == 0;
  return true;
}

__device__ __forceinline__ uint32_t lane_xor4(uint32_t x) { return dpp<0x1B>(dpp<kMirror8>(x)); }

// Lane a holds words w[k + 4 i] of chunk k (k in 0..3) for its side a / 4; a chunk is (i 0, side 0), (0, 1), (1, 0), (1, 1). Gives
// the lane chunks 2 (a / 4) and 2 (a / 4) + 1.
__device__ __forceinline__ void to_chunks(const uint32_t w[8], bool side, uint4 chunk[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t mine0 = side ? w[2 + k] : w[k], mine1 = side ? w[6 + k] : w[4 + k];
    const uint32_t other0 = lane_xor4(side ? w[k] : w[2 + k]), other1 = lane_xor4(side ? w[4 + k] : w[6 + k]);
    chunk[k] = uint4{side ? other0 : mine0, side ? mine0 : other0, side ? other1 : mine1, side ? mine1 : other1};
  }
}
__device__ __forceinline__ void from_chunks(uint32_t w[8], bool side, const uint4 chunk[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t mine0 = side ? chunk[k].y : chunk[k].x, mine1 = side ? chunk[k].w : chunk[k].z;
    const uint32_t other0 = lane_xor4(side ? chunk[k].x : chunk[k].y), other1 = lane_xor4(side ? chunk[k].z : chunk[k].w);
    w[k] = side ? other0 : mine0;
    w[2 + k] = side ? mine0 : other0;
    w[4 + k] = side ? other1 : mine1;
    w[6 + k] = side ? mine1 : other1;
  }
}
// Byte offset of a lane's first chunk in the half block, and between its two.
__device__ __forceinline__ int chunk_offset(int kind, int half, int a) {
  return kind ? kValueOffset + 256 * half + 16 * (8 * (a & 1) + 4 * (a >> 1 & 1) + 2 * (a >> 2)) : 256 * half + 128 * (a >> 2) + 16 * (a & 3);
}
__device__ __forceinline__ int chunk_stride(int kind) { return kind ? 16 : 64; }

// Eight waves a SIMD: 22 groups of a long prompt on each CU at once (89 registers and five waves: 2048 tokens 16.5 us, not 14.5).
__global__ __launch_bounds__(64 * kGroupWaves, 8) void kv_append_q4_groups_kernel(RowArgs args) {
  Group group;
  if (!group_of(args, group)) return;
  const int a = threadIdx.x % kRowLanes, h = threadIdx.x / kRowLanes % kKVHeads, kind = threadIdx.x / (kRowLanes * kKVHeads) % 2;
  const char* rows = (kind ? args.value + group.layer * args.value_layer : args.key + group.layer * args.key_layer) + h * (2 * kHeadDim) + 16 * a;
  const int64_t stride = kind ? args.value_token : args.key_token;
  half8_t x[kGroupTokens];
#pragma unroll
  for (int i = 0; i < kGroupTokens; ++i) {
    const int64_t token = group.token0 + i;
    x[i] = *reinterpret_cast<const half8_t*>(rows + stride * (token < 0 ? 0 : token < args.tokens ? token : args.tokens - 1));
  }
  char* const layer = args.pool + (static_cast<int64_t>(args.layer_begin + group.layer) * args.num_blocks * kKVHeads + h) * kUnitBytes;
  if (!group.whole) {
#pragma unroll
    for (int i = 0; i < kGroupTokens; ++i) {
      const int64_t slot = static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(group.slot >> 32), i))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(group.slot), i)));
      if (slot >= 0) store_row(layer + slot / kSlots * kBlockBytes, kind, static_cast<int>(slot % kSlots), a, quantize8(x[i]));
    }
    return;
  }
  uint32_t w[8], pair = 0;
#pragma unroll
  for (int i = 0; i < kGroupTokens; ++i) {
    const Levels q = quantize8(x[i]);
    w[i] = q.word;
    pair = a == i ? q.pair : pair;
  }
  if (kind != 0) {
    // Lanes a and a ^ 2 hold the low and the high halves of the same bytes. Each makes four columns' words: the bytes of a
    // token's even (u) and odd (v) levels, then four tokens of a column, in the order 0, 2, 1, 3.
    const bool upper = (a & 2) != 0;
    const uint32_t pick = upper ? 0x07030501u : 0x06020400u;
    uint32_t u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t other = dpp<kSwap2>(w[i]);
      const uint32_t low = upper ? other : w[i], high = upper ? w[i] : other;
      u[i] = (low & 0x0F0F0F0Fu) | (high << 4 & 0xF0F0F0F0u);
      v[i] = (low >> 4 & 0x0F0F0F0Fu) | (high & 0xF0F0F0F0u);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t u02 = __builtin_amdgcn_perm(u[4 * q + 2], u[4 * q], pick), u13 = __builtin_amdgcn_perm(u[4 * q + 3], u[4 * q + 1], pick);
      const uint32_t v02 = __builtin_amdgcn_perm(v[4 * q + 2], v[4 * q], pick), v13 = __builtin_amdgcn_perm(v[4 * q + 3], v[4 * q + 1], pick);
      w[4 * q] = __builtin_amdgcn_perm(u13, u02, 0x05040100u);
      w[4 * q + 1] = __builtin_amdgcn_perm(u13, u02, 0x07060302u);
      w[4 * q + 2] = __builtin_amdgcn_perm(v13, v02, 0x05040100u);
      w[4 * q + 3] = __builtin_amdgcn_perm(v13, v02, 0x07060302u);
    }
  }
  uint4 chunk[2];
  to_chunks(w, a >= 4, chunk);
  char* const unit = layer + group.first / kSlots * kBlockBytes;
  const int half = static_cast<int>(group.first / kGroupTokens % 2);
#pragma unroll
  for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(unit + chunk_offset(kind, half, a) + chunk_stride(kind) * k) = chunk[k];
  *reinterpret_cast<uint32_t*>(unit + pair_offset(kind, kGroupTokens * half + a)) = pair;
}

// The rows are whole lines that nothing reads soon, 9 MB and more of them: stored non-temporally 2048 tokens of 22 layers took 12.8 us
// instead of 15.1, 16384 71.9 instead of 95.4, and with a sum of K and V that reads them at once 27.6 instead of 30.0 and 182
// instead of 199. (Of the append's 13 MB of pool, which attention reads next, the same made 333 tokens slower, 5.0 to 5.4.)
__device__ __forceinline__ void store_past_caches(char* at, half8_t row) { __builtin_nontemporal_store(row, reinterpret_cast<half8_t*>(at)); }

__global__ __launch_bounds__(64 * kGroupWaves) void kv_read_q4_groups_kernel(RowArgs args) {
  Group group;
  if (!group_of(args, group)) return;
  const int a = threadIdx.x % kRowLanes, h = threadIdx.x / kRowLanes % kKVHeads, kind = threadIdx.x / (kRowLanes * kKVHeads) % 2;
  char* const rows = (kind ? args.value + group.layer * args.value_layer : args.key + group.layer * args.key_layer) + h * (2 * kHeadDim) + 16 * a;
  const int64_t stride = kind ? args.value_token : args.key_token;
  const char* const layer = args.pool + (static_cast<int64_t>(args.layer_begin + group.layer) * args.num_blocks * kKVHeads + h) * kUnitBytes;
  if (!group.whole) {
#pragma unroll
    for (int i = 0; i < kGroupTokens; ++i) {
      const int64_t slot = static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(group.slot >> 32), i))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(group.slot), i)));
      if (slot >= 0) {
        store_past_caches(rows + stride * (group.token0 + i), load_row(layer + slot / kSlots * kBlockBytes, kind, static_cast<int>(slot % kSlots), a));
      }
    }
    return;
  }
  const char* const unit = layer + group.first / kSlots * kBlockBytes;
  const int half = static_cast<int>(group.first / kGroupTokens % 2);
  uint4 chunk[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) chunk[k] = *reinterpret_cast<const uint4*>(unit + chunk_offset(kind, half, a) + chunk_stride(kind) * k);
  uint32_t pairs[kGroupTokens];  // the same of all eight lanes
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 four = *reinterpret_cast<const uint4*>(unit + pair_offset(kind, kGroupTokens * half + 4 * i));
    pairs[4 * i] = four.x;
    pairs[4 * i + 1] = four.y;
    pairs[4 * i + 2] = four.z;
    pairs[4 * i + 3] = four.w;
  }
  uint32_t w[8];
  from_chunks(w, a >= 4, chunk);
  if (kind != 0) {
    // The columns of lane a ^ 2, then the lane's half of every byte, and each token's eight levels as a K word.
    const bool upper = (a & 2) != 0;
    uint32_t n[2][8];  // of tokens 4 q + {0, 2, 1, 3}, column j
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t mine = w[4 * q + k], other = dpp<kSwap2>(mine);
        n[q][k] = (upper ? other >> 4 : mine) & 0x0F0F0F0Fu;
        n[q][4 + k] = (upper ? mine >> 4 : other) & 0x0F0F0F0Fu;
      }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int shift = t == 0 ? 0 : t == 1 ? 16 : t == 2 ? 8 : 24;
        float levels[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) levels[j] = static_cast<float>(n[q][j] >> shift & 255u);
        store_past_caches(rows + stride * (group.token0 + 4 * q + t), row_values(pair_low(pairs[4 * q + t]), pair_step(pairs[4 * q + t]), levels));
      }
  } else {
#pragma unroll
    for (int i = 0; i < kGroupTokens; ++i) {
      const uint32_t low = w[i] & 0x0F0F0F0Fu, high = w[i] >> 4 & 0x0F0F0F0Fu;  // j = 0 4 1 5 and 2 6 3 7
      float levels[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t from = (j & 2) != 0 ? high : low;
        levels[j] = static_cast<float>(from >> (8 * ((j >> 2) + 2 * (j & 1))) & 255u);
      }
      store_past_caches(rows + stride * (group.token0 + i), row_values(pair_low(pairs[i]), pair_step(pairs[i]), levels));
    }
  }
}

// Checks of both entry points; PC_OK with args filled in, or an error.
int row_args(RowArgs& args, const void* pool, int64_t num_blocks, int32_t layer_begin, int32_t num_layers, const void* key,
             int64_t key_layer_stride, int64_t key_token_stride, const void* value, int64_t value_layer_stride,
             int64_t value_token_stride, const int64_t* slot_mapping, int64_t num_tokens) {
  if (!pool || (num_tokens != 0 && (!key || !value || !slot_mapping))) return set_error(PC_ERR_ARGUMENT, "null pointer");
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
  args.begin = 0;
  args.layer_begin = layer_begin;
  return PC_OK;
}

bool rows_aligned(const RowArgs& args) {
  return aligned(args.key, 16) && aligned(args.value, 16) && args.key_layer % 16 == 0 && args.key_token % 16 == 0 &&
         args.value_layer % 16 == 0 && args.value_token % 16 == 0;
}

// Rows of one launch of the kernels that take a wave a token, and the launches that all rows take: one, but for more than 2^25
// tokens of a layer, or of several together, that are not 16-byte aligned.
constexpr uint32_t kLaunchRows = 1u << 28;
void launch_rows(void (*kernel)(RowArgs), RowArgs args, void* stream) {
  for (; args.begin < args.rows; args.begin += kLaunchRows) {
    const uint32_t rows = args.rows - args.begin < kLaunchRows ? args.rows - args.begin : kLaunchRows;
    hipLaunchKernelGGL(kernel, dim3((rows + kRowsPerGroup - 1) / kRowsPerGroup), dim3(kThreads), 0, static_cast<hipStream_t>(stream), args);
  }
}

// A wave a token and layer where there are few, for a short way to the end; eight tokens a wave above.
bool in_groups(const RowArgs& args) { return rows_aligned(args) && args.rows > kGroupRows; }
unsigned groups_grid_of(const RowArgs& args) {
  const uint64_t groups = (static_cast<uint64_t>(args.tokens) + 2 * kGroupTokens - 2) / kGroupTokens;
  return static_cast<unsigned>((groups * (args.rows / (args.tokens * 2 * kKVHeads)) + kGroupWaves - 1) / kGroupWaves);
}

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
  if (in_groups(args)) {
    hipLaunchKernelGGL(kv_append_q4_groups_kernel, dim3(groups_grid_of(args)), dim3(64 * kGroupWaves), 0, static_cast<hipStream_t>(stream), args);
    return check_launch("kv_append_q4");
  }
  launch_rows(rows_aligned(args) ? kv_append_q4_kernel<true> : kv_append_q4_kernel<false>, args, stream);
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
  if (in_groups(args)) {
    hipLaunchKernelGGL(kv_read_q4_groups_kernel, dim3(groups_grid_of(args)), dim3(64 * kGroupWaves), 0, static_cast<hipStream_t>(stream), args);
    return check_launch("kv_read_q4");
  }
  launch_rows(rows_aligned(args) ? kv_read_q4_kernel<true> : kv_read_q4_kernel<false>, args, stream);
  return check_launch("kv_read_q4");
}

}  // extern "C"
