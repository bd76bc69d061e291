// Paged decode attention over the 4-bit KV pool: one query token per sequence, one layer. The decode plan, the
// bins, the workspace, the part flags and the fault word are those of the fp16 kernel (pagedcore_hip.hip); the
// format of the pool is in q4_device.h.
//
// With rows k_t = lo_t + s_t n_t and v_t = lo'_t + s'_t n'_t, levels n in 0..15:
//   y_t = s_t (q . n_t) + lo_t sum(q),   p_t = exp((y_t - max y) / 8)
//   out = (sum_t (p_t s'_t) n'_t + sum_t p_t lo'_t) / sum_t p_t
// so scales and minima enter once per token and head, and the products run on the levels themselves:
//   * q . n on the fp16 instruction, n taken as the fp16 whose bits are n or 16 n (the subnormals n 2^-24 and n 2^-20:
//     exact, and one mask and at most one shift for two of them; the query's elements make up for the factor);
//   * (p s') n' on the bf16 instruction, n' as 16 + n' (bf16 bits 0x4180 | n' << 3, exact), p s' as bf16 and the bf16 of its
//     remainder in the two halves of the columns (16 bits of it; bf16 because p s' spans fp32's range), and
//     16 sum(p s') of the same rounded weights, from one more product with ones, is taken off at the end. 16 is the least
//     offset that needs no conversion: the sums hold three times what is wanted, 1.6 bits of their 24. (128 + n', a shift less in
//     eight levels, holds eighteen times it: outputs of 512 sequences of 2048 tokens whose values cancel, in steps of 1/8 to 1/4,
//     had an error of 4.6e-6, root mean square, instead of 1.1e-6.)
//
// One or two waves of a workgroup take a kv head of its bin, four blocks (64 tokens) a step. The row of a product's tile is
// chosen so that no data crosses lanes: tile i's row 4b + e is token 4i + e of the step's block b, which leaves lane
// (c, g) the scores of block g for head c % 8. The group has 8 query heads and a tile 16 columns (the heads twice), so
// the softmax takes tile 2a from columns 0-7 and tile 2a + 1 from columns 8-15: 32 tokens x 8 heads per four values
// of a lane, and each exponential is computed once.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "attn_plan.h"
#include "pagedcore_hip.h"
#include "pc_device.h"
#include "pc_internal.h"
#include "q4_device.h"

namespace {

using namespace attn_plan;
using namespace pc_device;
using pc_internal::aligned;
using pc_internal::check_launch;
using pc_internal::ok;
using pc_internal::set_error;
using q4_device::dpp;
using q4_device::kRotate8;
using q4_device::kUnitBytes;
using q4_device::pair_low;
using q4_device::pair_step;
using q4_device::kBlockBytes;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef int32_t int8_vt __attribute__((ext_vector_type(8), aligned(4)));

constexpr int kPartBytes = 2048 + 512;  // a wave's partial in LDS
// Partials a round trip (seven: 2048 tokens 8.3 us instead of 7.95, 64 ragged sequences 10.7 instead of 10.4, 32763 13.8 instead of 12.9).
// (Times in this file are of a call in a graph, launch interval included.)
constexpr int kMergeParts = 4;
// Bins of a group above which a long sequence's are spread over the XCDs. On one XCD its bins share 32 CUs, on all of them their
// partials meet in memory instead of in the L2. One call, us on one XCD / spread: 4096 tokens 8.9 / 9.5, 8192 11.1 / 10.3,
// six of 9000 14.3 / 13.4; 64 ragged sequences 10.4 / 13.1.
constexpr int kSpreadBins = 32;
constexpr int kStepBlocks = 4;
constexpr int64_t kMaxBlocks = 1 << 26;  // a block's place in a layer, in 128-byte lines, in 32 bits
static_assert(kMaxUnits == 256, "four vectors of block ids");
constexpr float kLazyLog2 = 8.0f;  // headroom (log2 of p) before the running max is raised

// Partial of one (sequence, kv head): lane (c, g) holds head c % 8, dims 16 T + 4 g + e, T = 2 (c / 8) + {0, 1}:
// unnormalized O, and the head's max (a base-2 exponent) and sum.
struct Part {
  float o[8];
  float m, l;
};

__device__ __forceinline__ float add_halves(float x) { return x + dpp<kRotate8>(x); }
__device__ __forceinline__ float max_halves(float x) { return fmaxf(x, dpp<kRotate8>(x)); }

// acc <- acc (+) p, the online-softmax fold.
__device__ __forceinline__ void fold_part(Part& acc, const Part& p) {
  const float mn = fmaxf(acc.m, p.m);
  const float so = exp2_fast(acc.m - mn);
  const float sn = exp2_fast(p.m - mn);
  acc.l = fmaf(p.l, sn, acc.l * so);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc.o[i] = fmaf(p.o[i], sn, acc.o[i] * so);
  acc.m = mn;
}

// A row's values may pass 65504 by half a step (row_values in q4_device.h), and so may their mean: it is 65504 then, by a minimum
// that hands a NaN on.
__device__ __forceinline__ void store_output(_Float16* rows, int lane, const Part& p) {
  const int c = lane & 15, g = lane >> 4;
  _Float16* at = rows + (c & 7) * kHeadDim + 32 * (c >> 3) + 4 * g;
  const float inverse = 1.0f / p.l;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    half4_t x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<_Float16>(p.o[4 * k + e] * inverse);
    const _Float16 most = static_cast<_Float16>(65504.f);
    *reinterpret_cast<half4_t*>(at + 16 * k) = __builtin_elementwise_minimum(x, half4_t{most, most, most, most});
  }
}

// A partial in a workspace slot: O in 2 KiB, then (m, l) of the 8 heads at 2048. Where the bins of a sequence run on one XCD,
// its L2 is where their partials meet, by plain stores and loads of 16 bytes (lane L's at 32 L); on several
// XCDs (SPREAD), whose L2s are not coherent with each other, by agent-scope ones of 8 bytes (at 8 L, 512 + 8 L, ...).
__device__ __forceinline__ void store_pair(char* at, float a, float b) {
  const uint64_t v = static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(at), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void load_pair(const char* at, float& a, float& b) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  a = __uint_as_float(static_cast<uint32_t>(v));
  b = __uint_as_float(static_cast<uint32_t>(v >> 32));
}
template <bool SPREAD>
__device__ __forceinline__ void store_part(char* slot, int lane, const Part& p) {
  if constexpr (SPREAD) {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_pair(slot + 512 * i + 8 * lane, p.o[2 * i], p.o[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<float4_t*>(slot + 32 * lane + 16 * i) = float4_t{p.o[4 * i], p.o[4 * i + 1], p.o[4 * i + 2], p.o[4 * i + 3]};
  }
  if (lane < kGroup) store_pair(slot + 2048 + 8 * lane, p.m, p.l);
}
template <bool SPREAD>
__device__ __forceinline__ Part load_part(const char* slot, int lane) {
  Part p;
  if constexpr (SPREAD) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_pair(slot + 512 * i + 8 * lane, p.o[2 * i], p.o[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4_t x = *reinterpret_cast<const float4_t*>(slot + 32 * lane + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) p.o[4 * i + e] = x[e];
    }
  }
  load_pair(slot + 2048 + 8 * (lane & 7), p.m, p.l);  // beside the flag, which has been polled: past the L1
  return p;
}

// A partial in LDS: O at 16 L and 1024 + 16 L of lane L, (m, l) at 2048 + 8 L.
__device__ __forceinline__ void put_part(char* area, int lane, const Part& p) {
  *reinterpret_cast<float4_t*>(area + 16 * lane) = float4_t{p.o[0], p.o[1], p.o[2], p.o[3]};
  *reinterpret_cast<float4_t*>(area + 1024 + 16 * lane) = float4_t{p.o[4], p.o[5], p.o[6], p.o[7]};
  reinterpret_cast<float*>(area + 2048)[2 * lane] = p.m;
  reinterpret_cast<float*>(area + 2048)[2 * lane + 1] = p.l;
}
__device__ __forceinline__ Part take_part(const char* area, int lane) {
  const float4_t a = *reinterpret_cast<const float4_t*>(area + 16 * lane), b = *reinterpret_cast<const float4_t*>(area + 1024 + 16 * lane);
  Part p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p.o[i] = a[i];
    p.o[4 + i] = b[i];
  }
  p.m = reinterpret_cast<const float*>(area + 2048)[2 * lane];
  p.l = reinterpret_cast<const float*>(area + 2048)[2 * lane + 1];
  return p;
}

// Eight levels of a word as fp16 subnormals: n 2^-24 for j = 0, 1, 4, 5 and, left where they are in the byte, n 2^-20 for
// j = 2, 3, 6, 7 (the query's elements make up for it, see scaled_query).
__device__ __forceinline__ half8_t key_levels(uint32_t w) {
  const uint32_t z = w >> 8;
  uint4_t r = {w & 0x000F000Fu, w & 0x00F000F0u, z & 0x000F000Fu, z & 0x00F000F0u};
  return __builtin_bit_cast(half8_t, r);
}

// Levels of two words (tokens 0-3 and 4-7; upper: the byte's upper half) as bf16 16 + n, n in bits 3-6 of each half. `bias` is
// 0x41804180 in a vector register: an and-or takes one constant from the scalar ones.
__device__ __forceinline__ bf16x8_t value_levels(uint32_t a, uint32_t b, bool upper, uint32_t bias) {
  constexpr uint32_t kLevels = 0x00780078u;
  uint4_t r = {((upper ? a >> 1 : a << 3) & kLevels) | bias, ((upper ? a >> 9 : a >> 5) & kLevels) | bias,
               ((upper ? b >> 1 : b << 3) & kLevels) | bias, ((upper ? b >> 9 : b >> 5) & kLevels) | bias};
  return __builtin_bit_cast(bf16x8_t, r);
}

// q with its elements j = 0, 1, 4, 5 of every eight times `even` and the others times `odd`.
__device__ __forceinline__ half8_t scaled_query(half8_t q, _Float16 even, _Float16 odd) {
  return q * half8_t{even, even, odd, odd, even, even, odd, odd};
}

__device__ __forceinline__ half8_t sixteenth_squared(half8_t q) {
  q *= static_cast<_Float16>(0.0625f);
  return q * q;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  bf16x2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float low_bf16(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_bf16(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// x with lanes 8-15 of each row of 16 replaced by lanes 0-7 of y (UPPER), or lanes 0-7 by lanes 8-15 of y.
template <bool UPPER>
__device__ __forceinline__ uint32_t take_half(uint32_t x, uint32_t y) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(x), static_cast<int>(y), kRotate8, 0xf, UPPER ? 0xc : 0x3, false));
}

// The largest of eight, none of them fresh from a matrix instruction. (fmaxf of values that the compiler cannot tell to be
// quiet costs an instruction each to make them so.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max8(const float (&y)[2][4]) {
  return max3(max3(max3(y[0][0], y[0][1], y[0][2]), y[0][3], y[1][0]), max3(y[1][1], y[1][2], y[1][3]), y[1][3]);
}

// The parts of one cut sequence that a bin waits for: first, first + stride, ... (count of them, at most 64).
// `spins`: how long; a level of the tree waits longer than all before it, which may have waited for a part that never came.
struct Waited {
  int first, stride, count, spins;
};

// A raised flag's low bits: the XCD where its part is to be seen; on all of them 1.
template <bool SPREAD>
__device__ __forceinline__ int flag_id() {
  if constexpr (SPREAD) return 1;
  else return xcc_id() + 1;
}

// Folds the waited parts into `total`, in order, as their flags rise, and lowers the flags. Returns PC_ATTN_FAULT_* bits.
template <bool SPREAD>
__device__ __forceinline__ int merge_parts(Part& total, char* slots, int slot0, const Waited& parts, int h, int lane, int key) {
  const int want = key | flag_id<SPREAD>();
  bool timeout = false, foreign = false;
  const int n = parts.count;
  if (n <= 0) return 0;
  // Lane k polls the flag of part k (lanes past the last one repeat it).
  int32_t* flag = reinterpret_cast<int32_t*>(part_slot(slots, slot0, parts.first + parts.stride * min(lane, n - 1), h) + kFlagOffset);
  int f = 0;
  for (int spins = 0; spins < parts.spins; ++spins) {
    f = __hip_atomic_load(flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_ballot_w64(!flag_of_call(f, key)) == 0) break;
    __builtin_amdgcn_s_sleep(1);
  }
  timeout = __builtin_amdgcn_ballot_w64(!flag_of_call(f, key)) != 0;
  foreign = __builtin_amdgcn_ballot_w64(flag_of_call(f, key) && f != want) != 0;
  asm volatile("" ::: "memory");
  // Past the last part it is loaded again and not folded.
#pragma nounroll
  for (int k = 0; k < n; k += kMergeParts) {
    Part p[kMergeParts];
#pragma unroll
    for (int i = 0; i < kMergeParts; ++i) p[i] = load_part<SPREAD>(part_slot(slots, slot0, parts.first + parts.stride * min(k + i, n - 1), h), lane);
#pragma unroll
    for (int i = 0; i < kMergeParts; ++i) {
      if (k + i < n) fold_part(total, p[i]);
    }
  }
  if (lane < n) __hip_atomic_store(flag, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (timeout || foreign) {
#pragma unroll
    for (int i = 0; i < 8; ++i) total.o[i] = NAN;
  }
  return (timeout ? PC_ATTN_FAULT_MERGE_TIMEOUT : 0) | (foreign ? PC_ATTN_FAULT_FOREIGN_XCD : 0);
}

// One step's bytes: four blocks of one head. The parts of the next step are loaded as this one's are used up.
struct Step {
  uint4_t k[2], v[2], kp[2], vp[2];

  __device__ __forceinline__ void load_keys(const char* kb) {
#pragma unroll
    for (int a = 0; a < 2; ++a) k[a] = *reinterpret_cast<const uint4_t*>(kb + 256 * a);
  }
  __device__ __forceinline__ void load_pairs(const char* vb, int c) {
#pragma unroll
    for (int a = 0; a < 2; ++a) kp[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::pair_offset(0, 8 * a + 4 * (c >> 3)));
#pragma unroll
    for (int a = 0; a < 2; ++a) vp[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::pair_offset(1, 8 * a + 4 * (c >> 3)));
  }
  __device__ __forceinline__ void load_values(const char* vb, int c) {
#pragma unroll
    for (int a = 0; a < 2; ++a) v[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::kValueOffset + 256 * a + 16 * c);
  }
};

// Where a lane finds its bytes of a step: its K row's chunk (of block c / 4 of the four) and block g's unit. Blocks past the
// segment's repeat its last one.
struct Blocks {
  const uint32_t* lines;  // of the segment's blocks in the layer, in units of 128 bytes (in LDS)
  int nblk;
  const char* lbase;
  int c, g;

  __device__ __forceinline__ void addresses(int u, const char*& kb, const char*& vb) const {
    kb = lbase + (static_cast<uint64_t>(lines[min(u + (c >> 2), nblk - 1)]) << 7) + 64 * (c & 3) + 16 * g;
    vb = lbase + (static_cast<uint64_t>(lines[min(u + g, nblk - 1)]) << 7);
  }
};

// PARTS waves a kv head, each its share of the bin's steps. With much to read it is bound by HBM: 256 sequences of 2048 tokens
// (151 MB) take 30.1 us with the launch, 5.0 TB/s (a large read: 6.3); vector instructions are half of that time. With little,
// by latency: 128 tokens 3.9 us, of which a launch that does nothing is 1.9, then record, rows, products in turn; a cut sequence
// adds its tree of partials (2048 tokens 7.9 us, 32763 13.1).
//   Two waves a head have more loads in flight and halve a bin's chain of steps: 256 sequences of 2048 tokens 30.1 us (one wave
// 37.2, four 31.0), 64 ragged ones 10.5 (11.1, 12.6), 256 of at most 64 tokens 8.6 (10.3, 8.0). One wave needs no barrier and no
// fold: 128 tokens 3.9 us (two 4.6), eight ragged sequences 7.8 (8.1), one of 8192 tokens 10.4 (10.9).
//   126 vector registers and no spills, of scalar ones neither, leave two workgroups of eight waves on a CU, which a plan of more
// bins than CUs needs (the build checks it).
template <bool APPEND, bool SPREAD, int PARTS>
__global__ __launch_bounds__(64 * PARTS * kKVHeads, 4) void paged_decode_q4_kernel(
    const int32_t* __restrict__ plan, const _Float16* query, char* pool, uint32_t num_blocks, int layer, int rows, int batch, int nslots,
    _Float16* out, char* workspace, const _Float16* new_key, const _Float16* new_value) {
  static_assert(PARTS == 1 || PARTS == 2, "a segment that goes on past a wave ends in the next");
  constexpr int kWaves = PARTS * kKVHeads;
  __shared__ uint32_t shared_lines[kWaves * kMaxUnits];
  __shared__ __attribute__((aligned(16))) char shared_parts[kWaves * 2 * kPartBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = wave % kKVHeads, part = wave / kKVHeads;
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  // The hardware deals consecutive workgroups to the XCDs in turn, and the plan's rows are in this order: a group of bins to
  // an XCD. SPREAD: consecutive workgroups take consecutive bins of one group.
  int row_index = static_cast<int>(blockIdx.x);
  if constexpr (SPREAD) {
    const uint32_t bins = gridDim.x / kGroups;
    row_index = static_cast<int>(blockIdx.x % bins * kGroups + blockIdx.x / bins);
    if (row_index >= rows) return;
  }
  const int32_t* row = plan + static_cast<int64_t>(row_index) * kRowInts;
  // The record (scalar loads) and the bin's block ids (lane L of vector k holds id 64 k + L) in one round trip: all of them are
  // wanted at one place, before any is looked at.
  int32_t idv[kMaxUnits / 64];
#pragma unroll
  for (int k = 0; k < kMaxUnits / 64; ++k) idv[k] = row[kRecordInts + 64 * k + lane];
  const int8_vt* fields = reinterpret_cast<const int8_vt*>(row);
  int8_vt header = fields[0], seg0 = fields[1], seg1 = fields[2], seg2 = fields[3], seg3 = fields[4];
  asm volatile("" : "+s"(header), "+s"(seg0), "+s"(seg1), "+s"(seg2), "+s"(seg3), "+v"(idv[0]), "+v"(idv[1]), "+v"(idv[2]), "+v"(idv[3]));
  const int nseg = header[0], nunits = header[1];
  if (nseg <= 0 || nseg > kMaxSegs || nunits <= 0 || nunits > kMaxUnits) return;  // padding rows do nothing
  // Field f of segment s.
  auto field = [&](int s, int f) {
    int v = seg0[f];
    v = s == 1 ? seg1[f] : v;
    v = s == 2 ? seg2[f] : v;
    return s == 3 ? seg3[f] : v;
  };
  // Its steps; a record whose segments are not its blocks does nothing.
  auto steps_of = [](int blocks) { return static_cast<int>(static_cast<uint32_t>(blocks + kStepBlocks - 1) / kStepBlocks); };
  const uint32_t n0 = seg0[3], n1 = nseg > 1 ? seg1[3] : 0, n2 = nseg > 2 ? seg2[3] : 0, n3 = nseg > 3 ? seg3[3] : 0;
  const uint32_t most = max(max(n0, n1), max(n2, n3)), least = min(min(n0, nseg > 1 ? n1 : n0), min(nseg > 2 ? n2 : n0, nseg > 3 ? n3 : n0));
  if (least == 0 || most > kMaxUnits || n0 + n1 + n2 + n3 != static_cast<uint32_t>(nunits)) return;
  const int steps = steps_of(n0) + steps_of(n1) + steps_of(n2) + steps_of(n3);
  // Each wave keeps the blocks' places for itself: no barrier before its first load. An id outside the pool is never
  // dereferenced (block 0 is read).
  uint32_t* const lines = shared_lines + wave * kMaxUnits;
  bool any_outside = false;
#pragma unroll
  for (int k = 0; k < kMaxUnits / 64; ++k) {
    if (64 * k < nunits) {
      const uint32_t id = static_cast<uint32_t>(idv[k]);
      any_outside |= __builtin_amdgcn_ballot_w64(id >= num_blocks && 64 * k + lane < nunits) != 0;
      lines[64 * k + lane] = (id >= num_blocks ? 0 : id) * static_cast<uint32_t>(kBlockBytes / 128);
    }
  }
  wave_lds_fence();
  char* const lbase = pool + static_cast<int64_t>(layer) * static_cast<int64_t>(num_blocks) * kBlockBytes + h * kUnitBytes;

  // This wave's steps [begin, end) of the bin's.
  const int begin = part * steps / PARTS, end = (part + 1) * steps / PARTS;

  // APPEND: lanes (c, g) quantise and store the new K (c < 8) and V row of segment g, if it ends its sequence and this wave has
  // its last step: the wave alone reads the unit, after this, and a wave's vector memory operations are done in order (the fence
  // keeps the compiler to it; a wait for the stores cost 0.3 us of 11.5 for 64 ragged sequences).
  if constexpr (APPEND) {
    int first = 0, sb = 0, len = 0, j0 = 0, nblk = 0, ends = 0;
#pragma unroll
    for (int s = 0, at = 0, step = 0; s < kMaxSegs; ++s) {
      const int n = s < nseg ? field(s, 3) : 0;
      step += steps_of(n);
      if (s == g) {
        first = at;
        sb = field(s, 0);
        len = field(s, 1);
        j0 = field(s, 2);
        nblk = n;
        ends = step;
      }
      at += n;
    }
    const int last = nblk > 0 ? first + nblk - 1 : 0;
    const bool mine = nblk > 0 && len > 0 && j0 + nblk == blocks_of(len) && sb >= 0 && sb < batch && ends > begin && ends <= end;
    const int a = c & 7, kind = c >> 3;
    const _Float16* src = (kind ? new_value : new_key) + (static_cast<int64_t>(mine ? sb : 0) * kKVHeads + h) * kHeadDim + 8 * a;
    const uint32_t line = lines[last];
    const bool in_pool = !any_outside || static_cast<uint32_t>(row[kRecordInts + last]) < num_blocks;
    if (__builtin_amdgcn_ballot_w64(mine) != 0) {
      const q4_device::Levels q = q4_device::quantize8(*reinterpret_cast<const half8_t*>(src));
      if (mine && in_pool) q4_device::store_row(lbase + (static_cast<uint64_t>(line) << 7), kind, (len - 1) % kSlots, a, q);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }

  uint32_t bias;
  asm("v_mov_b32 %0, 0x41804180" : "=v"(bias));
  // A zero that the compiler does not see through: p s + 0 is one instruction on the pair's half, p s a conversion and a product.
  float none;
  asm("s_mov_b32 %0, 0" : "=s"(none));
  char* const areas = shared_parts + wave * 2 * kPartBytes;
  // The wave's first and last segment, if it holds their first step but cannot write their rows by itself (-1: none): what
  // the wave did of them is in its first and second area.
  int first_seg = -1, last_seg = -1, first_end = 0, last_end = 0;
  bool first = true;
  int seg_begin = 0, seg_step = 0;
  for (int seg = 0; seg < nseg; ++seg) {
    const int sb = field(seg, 0), len = field(seg, 1), j0 = field(seg, 2), nblk = field(seg, 3), nspan = field(seg, 6);
    const int seg_steps = steps_of(nblk);
    const int from = max(begin - seg_step, 0), to = min(end - seg_step, seg_steps);
    if (from < to) {
      const Blocks at{lines + seg_begin, nblk, lbase, c, g};
      Step d;
      const char *kb, *vb;
      at.addresses(from * kStepBlocks, kb, vb);
      d.load_keys(kb);
      // Q of head c % 8, dims 8 g and 32 + 8 g on.
      const int qrow = sb < 0 || sb >= batch ? 0 : sb;
      const half8_t* src = reinterpret_cast<const half8_t*>(query + (static_cast<int64_t>(qrow) * kQHeads + kGroup * h + (c & 7)) * kHeadDim) + g;
      half8_t qa = src[0], qb = src[4];
      d.load_pairs(vb, c);
      d.load_values(vb, c);
      float m = 0.f, lsum = 0.f, usum = 0.f;
      float4_t acc[4], wacc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
      // (Set here, while the loads are on their way, and not behind the wait for them.)
      asm volatile("" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]), "+v"(wacc));
      // sum(q) of the lane's head, by a product with ones, and by another the sum of (q / 16)^2, which tells if the head may have
      // an element of 4096 or more (its square is past fp16's range; 4094, the next smaller one, gives 65472).
      // The products give 2^-20 (q . n) with 16 q at the places of n 2^-24; where 16 q might pass fp16's range 2^-24 (q . n) with
      // q / 16 at the others: what that rounds off, 2^-21 of an element of a head whose largest are thousands, is below the
      // sums' own roundings. `to_log2`: a score in this unit as a base-2 exponent, log2(e) / 8 over the unit.
      const _Float16 o = static_cast<_Float16>(1.f);
      const half8_t ones = {o, o, o, o, o, o, o, o};
      const float4_t zero = {0.f, 0.f, 0.f, 0.f};
      float4_t sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, qa, zero, 0, 0, 0);
      float4_t squares = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, sixteenth_squared(qa), zero, 0, 0, 0);
      sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, qb, sums, 0, 0, 0);
      squares = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, sixteenth_squared(qb), squares, 0, 0, 0);
      const bool large = !(squares[0] < 65500.f);
      const float qsum = sums[0] * (large ? 1.f / 16777216.f : 1.f / 1048576.f);
      const float to_log2 = large ? 16777216.f * kScoreToLog2 : 1048576.f * kScoreToLog2;
      const _Float16 even = static_cast<_Float16>(large ? 1.f : 16.f), odd = static_cast<_Float16>(large ? 0.0625f : 1.f);
      qa = scaled_query(qa, even, odd);
      qb = scaled_query(qb, even, odd);

      // One step, MORE: of which there is a next, whose loads go out behind the uses of the registers that they fill.
      auto one_step = [&](int x, auto more_steps) __attribute__((always_inline)) {
        constexpr bool MORE = decltype(more_steps)::value;
        const int u = x * kStepBlocks;
        if constexpr (MORE) at.addresses(u + kStepBlocks, kb, vb);
        float y[2][4];  // scores less the running max
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          float4_t even_tile = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(d.k[a][0]), qa, zero, 0, 0, 0);
          float4_t odd_tile = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(d.k[a][2]), qa, zero, 0, 0, 0);
          even_tile = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(d.k[a][1]), qb, even_tile, 0, 0, 0);
          odd_tile = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(d.k[a][3]), qb, odd_tile, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[a][e] = fmaf(pair_step(d.kp[a][e]), c < 8 ? even_tile[e] : odd_tile[e], fmaf(pair_low(d.kp[a][e]), qsum, -m));
          }
        }
        if constexpr (MORE) d.load_keys(kb);
        // Tokens of block u + g that exist; the score of one that does not is -inf and its weights are 0, whatever its bytes are.
        const int valid = u + g < nblk ? len - (j0 + u + g) * kSlots : 0;
        if (__builtin_amdgcn_ballot_w64(valid < kSlots) != 0) {
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool there = 8 * a + 4 * (c >> 3) + e < valid;
              y[a][e] = there ? y[a][e] : -INFINITY;
              d.vp[a][e] = there ? d.vp[a][e] : 0u;
            }
        }
        float bm = max8(y);
        if (x == from || __builtin_amdgcn_ballot_w64(bm * to_log2 > kLazyLog2) != 0) {
          bm = max_halves(max_over_groups(bm));  // of a first step finite: token 0 of its first block is valid
          if (x != from) {
            bm = fmaxf(bm, 0.f);
            const float alpha = exp2_fast(-bm * to_log2);
            lsum *= alpha;
            usum *= alpha;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][e] *= alpha;
#pragma unroll
            for (int e = 0; e < 4; ++e) wacc[e] *= alpha;
          }
          m += bm;
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[a][e] -= bm;
        }
        bf16x8_t weights[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_fast(y[a][e] * to_log2);
            lsum += p;
            w[e] = fmaf(p, pair_step(d.vp[a][e]), none);
            usum = fmaf(p, pair_low(d.vp[a][e]), usum);
          }
          const uint32_t hi0 = pack_bf16(w[0], w[1]), hi1 = pack_bf16(w[2], w[3]);
          const uint32_t lo0 = pack_bf16(w[0] - low_bf16(hi0), w[1] - high_bf16(hi0));
          const uint32_t lo1 = pack_bf16(w[2] - low_bf16(hi1), w[3] - high_bf16(hi1));
          // Columns 0-7: the weights of both tiles' tokens, columns 8-15 their remainders.
          const uint4_t wp = {take_half<true>(hi0, lo0), take_half<true>(hi1, lo1), take_half<false>(lo0, hi0), take_half<false>(lo1, hi1)};
          weights[a] = __builtin_bit_cast(bf16x8_t, wp);
        }
        if constexpr (MORE) d.load_pairs(vb, c);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value_levels(d.v[a][t >> 1], d.v[a][2 + (t >> 1)], (t & 1) != 0, bias), weights[a], acc[t], 0, 0, 0);
          }
          const uint4_t one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
          wacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, one), weights[a], wacc, 0, 0, 0);
        }
        if constexpr (MORE) d.load_values(vb, c);
      };
#pragma nounroll
      for (int x = from; x + 1 < to; ++x) one_step(x, std::true_type{});
      one_step(to - 1, std::false_type{});
      // A block id outside the pool among the segment's blocks here.
      bool bad = false;
      if (any_outside) {
#pragma unroll  // (a loop's stride and end would be held in scalar registers through the loops around, and spill others)
        for (int k = 0; k < kMaxUnits / 64; ++k) {
          const int u = kStepBlocks * from + lane + 64 * k;
          if (u < min(kStepBlocks * to, nblk)) bad |= static_cast<uint32_t>(row[kRecordInts + seg_begin + u]) >= num_blocks;
        }
        bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      }
      Part p;
      p.m = m * to_log2;
      p.l = add_halves(sum_over_groups(lsum));
      const float shift = fmaf(-16.f, add_halves(wacc[0]), add_halves(sum_over_groups(usum)));
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = add_halves(acc[k][e]), z = add_halves(acc[2 + k][e]);
          p.o[4 * k + e] = bad ? NAN : (c < 8 ? x : z) + shift;
        }
      if (from == 0 && to == seg_steps && nspan == 1) {
        if (sb >= 0 && sb < batch) store_output(out + (static_cast<int64_t>(sb) * kQHeads + kGroup * h) * kHeadDim, lane, p);
      } else {
        put_part(areas + (first ? 0 : kPartBytes), lane, p);
        if (from == 0) {
          first_seg = first ? seg : first_seg;
          first_end = first ? seg_step + seg_steps : first_end;
          last_seg = first ? last_seg : seg;
          last_end = first ? last_end : seg_step + seg_steps;
        }
      }
      first = false;
    }
    seg_begin += nblk;
    seg_step += seg_steps;
  }
  int fault = any_outside ? PC_ATTN_FAULT_BLOCK_ID : 0;
  if constexpr (PARTS > 1) __syncthreads();
  else wave_lds_fence();
  char* const slots = workspace + kWorkspaceHeader;
  const int key = flag_key(row[2], layer);
  int tail_lane = lane;  // what is computed from it below is not carried through the loop above
  asm volatile("" : "+v"(tail_lane));
  // The later segment first: another bin may wait for its part, and the bin's first segment may have to wait itself.
#pragma nounroll
  for (int r = 1; r >= 0; --r) {
    const int seg = r ? last_seg : first_seg;
    if (seg < 0) continue;
    const int8_vt again = fields[1 + seg];  // what the loop does not use of it has not been kept
    const int sb = again[0], kidx = again[5], nspan = again[6], slot0 = again[7], k00 = again[4];
    const int seg_end = r ? last_end : first_end;
    Part total = take_part(areas + r * kPartBytes, tail_lane);
    // The wave behind this one, if this is its first segment.
    if (part + 1 < PARTS && end < seg_end) fold_part(total, take_part(areas + kKVHeads * 2 * kPartBytes, tail_lane));
    bool last = true;
    if (nspan != 1) {
      // The span's slots [slot0, slot0 + parts - 1) lie in the workspace, and the part in the span.
      if (slot0 < 0 || nspan < 2 || slot0 + static_cast<int64_t>(nspan) - 1 > nslots || kidx < 0 || kidx >= nspan || k00 < 0 ||
          k00 + static_cast<int64_t>(kGroups) * kidx != row_index) {
        continue;
      }
      last = kidx == nspan - 1;
      // A tree: at every level the last part of 2^bits (and the span's last part) folds the others', by now of 2^bits times as
      // many parts each. A level costs a flag's way and one trip for every kMergeParts partials: of many parts, which are
      // spread, four at a time are best (32763 tokens, 256 parts: 12.9 us; eight 14.5, sixteen 15.6); of up to 32 eight (4096
      // tokens, 32 parts on one XCD: 8.9 us; four 9.2, sixteen 9.6), and up to sixteen at once (8 ragged sequences: 7.85 us;
      // four 8.2, eight 8.8). By the parts alone: SPREAD goes by the plan's rows, padding among them, and the order of the
      // sums, so the output's bits, must not.
      const int bits = nspan > kSpreadBins ? 2 : (nspan > 16 ? 3 : 4), others = (1 << bits) - 1;
#pragma nounroll
      for (int shift = 0, at = kidx, spins = kMaxSpins; at > 0 && (last || (at & others) == others); shift += bits, at >>= bits, spins = min(2 * spins, 16 * kMaxSpins)) {
        const Waited waited = {(((at & ~others) + 1) << shift) - 1, 1 << shift, at & others, spins};
        fault |= merge_parts<SPREAD>(total, slots, slot0, waited, h, tail_lane, key);
      }
    }
    if (last) {
      if (sb >= 0 && sb < batch) store_output(out + (static_cast<int64_t>(sb) * kQHeads + kGroup * h) * kHeadDim, tail_lane, total);
    } else {
      char* slot = part_slot(slots, slot0, kidx, h);
      store_part<SPREAD>(slot, tail_lane, total);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (tail_lane == 0) {
        __hip_atomic_store(reinterpret_cast<int32_t*>(slot + kFlagOffset), key | flag_id<SPREAD>(), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (fault != 0 && tail_lane == 0) {
    __hip_atomic_fetch_or(reinterpret_cast<int32_t*>(workspace), fault, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

template <bool APPEND>
int launch(void* out, const void* query, void* pool, int64_t num_blocks, int32_t layer, const int32_t* context_lens, int32_t batch,
           int32_t max_blocks, const int32_t* plan, int32_t num_records, const void* new_key, const void* new_value,
           void* workspace, void* stream) {
  if (!pool || (num_records != 0 && !plan)) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (batch != 0 && (!out || !query || !context_lens || (APPEND && (!new_key || !new_value)))) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (!workspace) return set_error(PC_ERR_ARGUMENT, "workspace required (null pointer)");
  if (num_blocks < 1 || num_blocks > kMaxBlocks) return set_error(PC_ERR_ARGUMENT, "num_blocks out of range [1, 2^26]");
  if (layer < 0 || layer >= kLayers) return set_error(PC_ERR_ARGUMENT, "layer %d outside [0, 22)", layer);
  if (int rc = check_attn_shape(batch, max_blocks)) return rc;
  if (!aligned(query, 16) || !aligned(out, 16) || !aligned(pool, 128) || !aligned(workspace, 256) || !aligned(plan, 16) ||
      !aligned(context_lens, 4) || !aligned(new_key, 16) || !aligned(new_value, 16)) {
    return set_error(PC_ERR_ARGUMENT, "query/out/plan/new rows must be 16-byte, pool 128-byte, workspace 256-byte aligned");
  }
  if (int rc = check_plan_rows(num_records, batch, max_blocks, 2 * 64 * kKVHeads)) return rc;
  if (batch == 0 || num_records == 0) return ok();
  // Fewer bins a group, or of a sequence, and each of an XCD's CUs has at most two of them. Rows of a padded plan count, so that
  // behind a wide table short sequences are spread too, which costs time (13.1 us for 10.4 above) and changes no bit.
  const bool spread = num_records > kGroups * kSpreadBins && max_blocks > kMinBinBlocks * kSpreadBins;
  // Bins of one segment and, at their least, two steps.
  const bool single = batch <= kGroups && static_cast<int64_t>(batch) * max_blocks <= kTargetBins * kMinBinBlocks;
  const auto kernel = spread ? (single ? paged_decode_q4_kernel<APPEND, true, 1> : paged_decode_q4_kernel<APPEND, true, 2>)
                             : (single ? paged_decode_q4_kernel<APPEND, false, 1> : paged_decode_q4_kernel<APPEND, false, 2>);
  const unsigned grid = static_cast<unsigned>(spread ? (num_records + kGroups - 1) / kGroups * kGroups : num_records);
  (void)hipGetLastError();
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * kKVHeads * (single ? 1 : 2)), 0,
                     static_cast<hipStream_t>(stream), plan, static_cast<const _Float16*>(query), static_cast<char*>(pool), static_cast<uint32_t>(num_blocks),
                     layer, num_records, batch, static_cast<int>(slots_bound(batch, max_blocks)), static_cast<_Float16*>(out),
                     static_cast<char*>(workspace), static_cast<const _Float16*>(new_key), static_cast<const _Float16*>(new_value));
  return check_launch(APPEND ? "kv_append_paged_decode_q4" : "paged_decode_q4");
}

}  // namespace

extern "C" {

int pc_paged_decode_attn_q4(void* out, const void* query, const void* pool, int64_t num_blocks, int32_t layer,
                            const int32_t* context_lens, int32_t batch, int32_t max_blocks, const int32_t* plan,
                            int32_t num_records, void* workspace, void* stream) {
  return launch<false>(out, query, const_cast<void*>(pool), num_blocks, layer, context_lens, batch, max_blocks, plan, num_records,
                       nullptr, nullptr, workspace, stream);
}

int pc_kv_append_paged_decode_attn_q4(void* out, const void* query, void* pool, int64_t num_blocks, int32_t layer,
                                      const int32_t* context_lens, int32_t batch, int32_t max_blocks, const int32_t* plan,
                                      int32_t num_records, const void* new_key, const void* new_value, void* workspace,
                                      void* stream) {
  return launch<true>(out, query, pool, num_blocks, layer, context_lens, batch, max_blocks, plan, num_records, new_key, new_value,
                      workspace, stream);
}

}  // extern "C"
