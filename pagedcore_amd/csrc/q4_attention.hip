// Paged decode attention over the 4-bit KV pool: one query token per sequence, one layer. The decode plan, the
// bins, the workspace, the part flags and the fault word are those of the fp16 kernel (pagedcore_hip.hip); the
// format of the pool is in q4_device.h.
//
// With rows k_t = lo_t + s_t n_t and v_t = lo'_t + s'_t n'_t, levels n in 0..15:
//   y_t = s_t (q . n_t) + lo_t sum(q),   p_t = exp((y_t - max y) / 8)
//   out = (sum_t (p_t s'_t) n'_t + sum_t p_t lo'_t) / sum_t p_t
// so scales and minima enter once per token and head, and the products run on the levels themselves:
//   * q . n on the fp16 instruction, n taken as the fp16 whose bits are n (the subnormal n 2^-24: exact, and one
//     mask and shift for two of them);
//   * (p s') n' on the bf16 instruction, n' as 128 + n' (bf16 bits 0x4300 | n'), p s' as bf16 and the bf16 of its
//     remainder in the two halves of the columns (16 bits of it; bf16 because p s' spans fp32's range), and
//     128 sum(p s') of the same rounded weights, from one more product with ones, is taken off at the end.
//
// Each of the four waves of a workgroup takes one kv head of its bin, four blocks (64 tokens) a step. The row of a
// product's tile is chosen so that no data crosses lanes: tile i's row 4b + e is token 4i + e of the step's block
// b, which leaves lane (c, g) the scores of block g for one head. The group has 8 query heads and a tile 16
// columns, so two tiles share an accumulator: columns 0-7 hold the heads for tile 2a, columns 8-15 for tile
// 2a + 1 (the operand's other half is zero), and the softmax runs on 32 tokens x 8 heads per four values of a lane.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

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
using q4_device::kBlockBytes;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 64 * kKVHeads;
constexpr int kStepBlocks = 4;
// A raw score, in units of 2^-24, to a base-2 exponent: 2^24 log2(e) / 8.
constexpr float kRawToLog2 = 16777216.0f * kScoreToLog2;
constexpr float kLazyLog2 = 8.0f;  // headroom (log2 of p) before the running max is raised

// Partial of one (sequence, kv head): lane (c, g) holds head c % 8, dims 16 T + 4 g + e, T = 2 (c / 8) + {0, 1}:
// unnormalized O, and the head's max (raw) and sum.
struct Part {
  float o[8];
  float m, l;
};

__device__ __forceinline__ float add_halves(float x) { return x + dpp<kRotate8>(x); }
__device__ __forceinline__ float max_halves(float x) { return fmaxf(x, dpp<kRotate8>(x)); }

// acc <- acc (+) p, the online-softmax fold.
__device__ __forceinline__ void fold_part(Part& acc, const Part& p) {
  const float mn = fmaxf(acc.m, p.m);
  const float so = exp2_fast((acc.m - mn) * kRawToLog2);
  const float sn = exp2_fast((p.m - mn) * kRawToLog2);
  acc.l = fmaf(p.l, sn, acc.l * so);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc.o[i] = fmaf(p.o[i], sn, acc.o[i] * so);
  acc.m = mn;
}

__device__ __forceinline__ void store_output(_Float16* rows, int lane, const Part& p) {
  const int c = lane & 15, g = lane >> 4;
  _Float16* at = rows + (c & 7) * kHeadDim + 32 * (c >> 3) + 4 * g;
  const float inverse = 1.0f / p.l;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    half4_t x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<_Float16>(p.o[4 * k + e] * inverse);
    *reinterpret_cast<half4_t*>(at + 16 * k) = x;
  }
}

// A partial in a workspace slot: lane L's O at byte 32 L, then (m, l) of the 8 heads at 2048.
__device__ __forceinline__ void store_part(char* slot, int lane, const Part& p) {
  float4_t* d = reinterpret_cast<float4_t*>(slot + lane * 32);
  d[0] = float4_t{p.o[0], p.o[1], p.o[2], p.o[3]};
  d[1] = float4_t{p.o[4], p.o[5], p.o[6], p.o[7]};
  if (lane < kGroup) {
    reinterpret_cast<float*>(slot + 2048)[2 * lane] = p.m;
    reinterpret_cast<float*>(slot + 2048)[2 * lane + 1] = p.l;
  }
}

__device__ __forceinline__ Part load_part(const char* slot, int lane) {
  const float4_t* d = reinterpret_cast<const float4_t*>(slot + lane * 32);
  const float4_t a = d[0], b = d[1];
  const float* e = reinterpret_cast<const float*>(slot + 2048) + 2 * (lane & 7);
  Part p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p.o[i] = a[i];
    p.o[4 + i] = b[i];
  }
  // The flag shares this line and has been polled: read past the L1.
  p.m = __hip_atomic_load(e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  p.l = __hip_atomic_load(e + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return p;
}

// Eight levels of a word as fp16 subnormals n 2^-24.
__device__ __forceinline__ half8_t key_levels(uint32_t w) {
  uint4_t r = {w & 0x000F000Fu, w >> 4 & 0x000F000Fu, w >> 8 & 0x000F000Fu, w >> 12 & 0x000F000Fu};
  return __builtin_bit_cast(half8_t, r);
}

// Levels of two words (tokens 0-3 and 4-7; `high`: the byte's upper half) as bf16 128 + n.
__device__ __forceinline__ bf16x8_t value_levels(uint32_t a, uint32_t b, int shift) {
  uint4_t r = {(a >> shift & 0x000F000Fu) | 0x43004300u, (a >> (8 + shift) & 0x000F000Fu) | 0x43004300u,
               (b >> shift & 0x000F000Fu) | 0x43004300u, (b >> (8 + shift) & 0x000F000Fu) | 0x43004300u};
  return __builtin_bit_cast(bf16x8_t, r);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  bf16x2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float low_bf16(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_bf16(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ float pair_low(uint32_t x) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x))); }
__device__ __forceinline__ float pair_step(uint32_t x) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x >> 16))); }

// x with lanes 8-15 of each row of 16 replaced by lanes 0-7 of y (UPPER), or lanes 0-7 by lanes 8-15 of y.
template <bool UPPER>
__device__ __forceinline__ uint32_t take_half(uint32_t x, uint32_t y) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(x), static_cast<int>(y), kRotate8, 0xf, UPPER ? 0xc : 0x3, false));
}

template <bool APPEND>
__global__ __launch_bounds__(kThreads) void paged_decode_q4_kernel(const int32_t* plan, const _Float16* query, char* pool,
                                                                  int64_t num_blocks, int layer, int batch, int nslots,
                                                                  _Float16* out, char* workspace, const _Float16* new_key,
                                                                  const _Float16* new_value) {
  const int h = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int32_t* row = plan + static_cast<int64_t>(blockIdx.x) * kRowInts;
  const int32_t* ids = row + kRecordInts;
  char* const slots = workspace + kWorkspaceHeader;
  int32_t rec[kRecordInts];
#pragma unroll
  for (int i = 0; i < kRecordInts; ++i) rec[i] = row[i];
  const int nseg = rec[0], nunits = rec[1];
  if (nseg <= 0 || nseg > kMaxSegs || nunits <= 0 || nunits > kMaxUnits) return;  // padding rows do nothing
  const int key = flag_key(rec[2], layer);
  char* const lbase = pool + static_cast<int64_t>(layer) * num_blocks * kBlockBytes + h * kUnitBytes;

  auto field = [&](int s, int f) {
    return s == 0 ? rec[8 + f] : s == 1 ? rec[16 + f] : s == 2 ? rec[24 + f] : rec[32 + f];
  };

  // APPEND: lanes (c, g) quantise and store the new K (c < 8) and V row of segment g, if the bin holds its sequence's last
  // block, before this wave (which alone reads the unit) reads it: a wave's memory operations are done in order.
  if constexpr (APPEND) {
    int first = 0, sb = 0, len = 0, j0 = 0, nblk = 0;
#pragma unroll
    for (int s = 0, at = 0; s < kMaxSegs; ++s) {
      if (s == g) {
        first = at;
        sb = field(s, 0);
        len = field(s, 1);
        j0 = field(s, 2);
        nblk = field(s, 3);
      }
      at += max(field(s, 3), 1);
    }
    const int last = first + nblk - 1;
    const bool mine = g < nseg && nblk > 0 && len > 0 && j0 + nblk == blocks_of(len) && sb >= 0 && sb < batch && last < nunits;
    const uint32_t id = static_cast<uint32_t>(ids[mine ? last : 0]);
    const int a = c & 7, kind = c >> 3;
    const _Float16* src = (kind ? new_value : new_key) + (static_cast<int64_t>(mine ? sb : 0) * kKVHeads + h) * kHeadDim + 8 * a;
    const q4_device::Levels q = q4_device::quantize8(*reinterpret_cast<const half8_t*>(src));
    if (mine && id < static_cast<uint64_t>(num_blocks)) {
      q4_device::store_row(lbase + static_cast<int64_t>(id) * kBlockBytes, kind, (len - 1) % kSlots, a, q);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  Part first_part, last_part;
  bool any_bad = false;
  int seg = 0, seg_end = 0;
  for (; seg < nseg; ++seg) {
    const int seg_begin = seg_end;
    const int sb = field(seg, 0), len = field(seg, 1), j0 = field(seg, 2), nblk = field(seg, 3), nspan = field(seg, 6);
    seg_end = seg_begin + max(nblk, 1);
    if (nblk <= 0 || seg_end > nunits) break;  // malformed record
    // Q of head c % 8 in the columns of the first (c < 8) or of the second tile of a pair; sum(q) 2^-24.
    const int qb = sb < 0 || sb >= batch ? 0 : sb;
    const half8_t* src = reinterpret_cast<const half8_t*>(query + (static_cast<int64_t>(qb) * kQHeads + kGroup * h + (c & 7)) * kHeadDim) + g;
    const half8_t qa = src[0], qb8 = src[4];
    const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
    const half8_t q0a = c < 8 ? qa : none, q0b = c < 8 ? qb8 : none, q1a = c < 8 ? none : qa, q1b = c < 8 ? none : qb8;
    float qsum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) qsum += static_cast<float>(qa[j]) + static_cast<float>(qb8[j]);
    qsum = sum_over_groups(qsum) * (1.0f / 16777216.0f);

    float m = 0.f, lsum = 0.f, usum = 0.f;
    float4_t acc[4], wacc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
    bool bad = false;

    for (int u = 0; u < nblk; u += kStepBlocks) {
      const uint32_t idk = static_cast<uint32_t>(ids[seg_begin + min(u + (c >> 2), nblk - 1)]);
      const uint32_t idv = static_cast<uint32_t>(ids[seg_begin + min(u + g, nblk - 1)]);
      const bool out_of_pool = idv >= static_cast<uint64_t>(num_blocks);
      bad |= __builtin_amdgcn_ballot_w64(out_of_pool) != 0;
      // never dereferenced out of the pool
      const char* kb = lbase + static_cast<int64_t>(idk >= static_cast<uint64_t>(num_blocks) ? 0 : idk) * kBlockBytes + 64 * (c & 3) + 16 * g;
      const char* vb = lbase + static_cast<int64_t>(out_of_pool ? 0 : idv) * kBlockBytes;
      uint4_t kw[2], vw[2], kp[2], vp[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        kw[a] = *reinterpret_cast<const uint4_t*>(kb + 256 * a);
        vw[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::kValueOffset + 256 * a + 16 * c);
        kp[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::pair_offset(0, 8 * a + 4 * (c >> 3)));
        vp[a] = *reinterpret_cast<const uint4_t*>(vb + q4_device::pair_offset(1, 8 * a + 4 * (c >> 3)));
      }
      float y[2][4];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float4_t s = {0.f, 0.f, 0.f, 0.f};
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(kw[a][0]), q0a, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(kw[a][1]), q0b, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(kw[a][2]), q1a, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_levels(kw[a][3]), q1b, s, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[a][e] = fmaf(pair_low(kp[a][e]), qsum, pair_step(kp[a][e]) * s[e]);
      }
      // Tokens of block u + g that exist; the score of one that does not is -inf and its weights are 0, whatever its bytes are.
      const int valid = u + g < nblk ? len - (j0 + u + g) * kSlots : 0;
      const bool full = __builtin_amdgcn_ballot_w64(valid < kSlots) == 0;
      if (!full) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[a][e] = 8 * a + 4 * (c >> 3) + e < valid ? y[a][e] : -INFINITY;
      }
      const float bm = fmaxf(fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[0][2], y[0][3])), fmaxf(fmaxf(y[1][0], y[1][1]), fmaxf(y[1][2], y[1][3])));
      if (u == 0) {
        m = max_halves(max_over_groups(bm));  // token 0 of the first block is valid
      } else if (__builtin_amdgcn_ballot_w64((bm - m) * kRawToLog2 > kLazyLog2) != 0) {
        const float mn = fmaxf(m, max_halves(max_over_groups(bm)));
        const float alpha = exp2_fast((m - mn) * kRawToLog2);
        lsum *= alpha;
        usum *= alpha;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] *= alpha;
#pragma unroll
        for (int e = 0; e < 4; ++e) wacc[e] *= alpha;
        m = mn;
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp2_fast((y[a][e] - m) * kRawToLog2);
          lsum += p;
          float low = pair_low(vp[a][e]);
          w[e] = p * pair_step(vp[a][e]);
          if (!full && 8 * a + 4 * (c >> 3) + e >= valid) low = w[e] = 0.f;
          usum = fmaf(p, low, usum);
        }
        const uint32_t hi0 = pack_bf16(w[0], w[1]), hi1 = pack_bf16(w[2], w[3]);
        const uint32_t lo0 = pack_bf16(w[0] - low_bf16(hi0), w[1] - high_bf16(hi0));
        const uint32_t lo1 = pack_bf16(w[2] - low_bf16(hi1), w[3] - high_bf16(hi1));
        // Columns 0-7: the weights of both tiles' tokens, columns 8-15 their remainders.
        const uint4_t wp = {take_half<true>(hi0, lo0), take_half<true>(hi1, lo1), take_half<false>(lo0, hi0), take_half<false>(lo1, hi1)};
        const bf16x8_t weights = __builtin_bit_cast(bf16x8_t, wp);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value_levels(vw[a][t >> 1], vw[a][2 + (t >> 1)], 4 * (t & 1)), weights, acc[t], 0, 0, 0);
        }
        const uint4_t one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
        wacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, one), weights, wacc, 0, 0, 0);
      }
    }
    Part p;
    p.m = m;
    p.l = add_halves(sum_over_groups(lsum));
    const float shift = fmaf(-128.f, add_halves(wacc[0]), add_halves(sum_over_groups(usum)));
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = add_halves(acc[k][e]), z = add_halves(acc[2 + k][e]);
        p.o[4 * k + e] = bad ? NAN : (c < 8 ? x : z) + shift;
      }
    any_bad |= bad;
    if (nspan == 1) {
      if (sb >= 0 && sb < batch) {
        store_output(out + (static_cast<int64_t>(sb) * kQHeads + kGroup * h) * kHeadDim, lane, p);
      }
    } else {
      if (seg == 0) first_part = p;
      if (seg == nseg - 1) last_part = p;
    }
  }
  const bool complete = seg == nseg && seg_end == nunits;  // the record's segments cover its blocks

  const int b0 = rec[8], k00 = rec[12], kidx0 = rec[13], nspan0 = rec[14], slot0 = rec[15];
  const int sl = nseg - 1;
  const int kidxl = field(sl, 5), nspanl = field(sl, 6), slotl = field(sl, 7);
  // The span's slots [first, first + parts - 1) lie in the workspace.
  auto slots_ok = [&](int first, int parts) { return first >= 0 && parts >= 2 && first + static_cast<int64_t>(parts) - 1 <= nslots; };

  // A part that is not the last of its span: store it, wait for the acknowledgement, then raise its flag.
  if (complete && nspanl > 1 && kidxl < nspanl - 1 && kidxl >= 0 && slots_ok(slotl, nspanl)) {
    char* slot = part_slot(slots, slotl, kidxl, h);
    store_part(slot, lane, last_part);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (lane == 0) {
      __hip_atomic_store(reinterpret_cast<int32_t*>(slot + kFlagOffset), key | (xcc_id() + 1), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  int fault = any_bad ? PC_ATTN_FAULT_BLOCK_ID : 0;
  // The last part of a cut sequence: the other parts in order as their flags rise, and this bin's part last. The bins of a
  // sequence run on one XCD, whose L2 their partials meet in; the earlier ones were dispatched first and wait for nothing.
  if (complete && nspan0 > 1 && kidx0 == nspan0 - 1 && slots_ok(slot0, nspan0) &&
      k00 + static_cast<int64_t>(kGroups) * kidx0 == static_cast<int64_t>(blockIdx.x) && k00 >= 0) {
    const int want = key | (xcc_id() + 1);
    bool timeout = false, foreign = false;
    Part total;
#pragma unroll
    for (int i = 0; i < 8; ++i) total.o[i] = 0.f;
    total.m = -INFINITY;
    total.l = 0.f;
    for (int k = 0; k < nspan0 - 1; ++k) {
      const char* slot = part_slot(slots, slot0, k, h);
      int f = 0;
      for (int spins = 0; spins < kMaxSpins && !timeout; ++spins) {
        f = __builtin_amdgcn_readfirstlane(
            __hip_atomic_load(reinterpret_cast<const int32_t*>(slot + kFlagOffset), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        if (flag_of_call(f, key)) break;
        __builtin_amdgcn_s_sleep(2);
      }
      timeout |= !flag_of_call(f, key);
      foreign |= flag_of_call(f, key) && f != want;  // raised on another XCD: its partial is not visible here
      asm volatile("" ::: "memory");
      fold_part(total, load_part(slot, lane));
    }
    fold_part(total, first_part);
    if (timeout || foreign) {
#pragma unroll
      for (int i = 0; i < 8; ++i) total.o[i] = NAN;
      fault |= (timeout ? PC_ATTN_FAULT_MERGE_TIMEOUT : 0) | (foreign ? PC_ATTN_FAULT_FOREIGN_XCD : 0);
    }
    for (int k = lane; k < nspan0 - 1; k += 64) {
      __hip_atomic_store(reinterpret_cast<int32_t*>(part_slot(slots, slot0, k, h) + kFlagOffset), 0, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    }
    if (b0 >= 0 && b0 < batch) store_output(out + (static_cast<int64_t>(b0) * kQHeads + kGroup * h) * kHeadDim, lane, total);
  }
  if (fault != 0 && lane == 0) {
    __hip_atomic_fetch_or(reinterpret_cast<int32_t*>(workspace), fault, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

template <bool APPEND>
int launch(void* out, const void* query, void* pool, int64_t num_blocks, int32_t layer, const int32_t* context_lens, int32_t batch,
           int32_t max_blocks, const int32_t* plan, int32_t num_records, const void* new_key, const void* new_value,
           void* workspace, void* stream) {
  if (!out || !query || !pool || !context_lens || !plan) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (APPEND && (!new_key || !new_value)) return set_error(PC_ERR_ARGUMENT, "null pointer");
  if (!workspace) return set_error(PC_ERR_ARGUMENT, "workspace required (null pointer)");
  if (num_blocks < 1 || num_blocks > INT32_MAX) return set_error(PC_ERR_ARGUMENT, "num_blocks out of range");
  if (layer < 0 || layer >= kLayers) return set_error(PC_ERR_ARGUMENT, "layer %d outside [0, 22)", layer);
  if (int rc = check_attn_shape(batch, max_blocks)) return rc;
  if (!aligned(query, 16) || !aligned(out, 16) || !aligned(pool, 128) || !aligned(workspace, 256) || !aligned(plan, 16) ||
      !aligned(context_lens, 4) || !aligned(new_key, 16) || !aligned(new_value, 16)) {
    return set_error(PC_ERR_ARGUMENT, "query/out/plan/new rows must be 16-byte, pool 128-byte, workspace 256-byte aligned");
  }
  if (num_records < 0 || num_records > plan_rows_bound(batch, max_blocks)) {
    return set_error(PC_ERR_ARGUMENT, "num_records %d outside [0, pc_attn_plan_capacity]", num_records);
  }
  if (batch == 0 || num_records == 0) return ok();
  (void)hipGetLastError();
  hipLaunchKernelGGL(paged_decode_q4_kernel<APPEND>, dim3(static_cast<unsigned>(num_records)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), plan, static_cast<const _Float16*>(query), static_cast<char*>(pool), num_blocks,
                     layer, batch, static_cast<int>(slots_bound(batch, max_blocks)), static_cast<_Float16*>(out),
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
