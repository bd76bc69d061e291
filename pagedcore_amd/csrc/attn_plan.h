// The decode plan's rows, the workspace's partial slots and their flags, shared by the paged decode
// attention kernels of the fp16 and of the 4-bit pool (not part of the C ABI): one plan and one
// workspace serve both.
#ifndef PAGEDCORE_ATTN_PLAN_H
#define PAGEDCORE_ATTN_PLAN_H

#include <hip/hip_runtime.h>

#include <algorithm>

#include <stdint.h>

#include "pagedcore_hip.h"
#include "pc_internal.h"

namespace attn_plan {

constexpr int kLayers = 22;
constexpr int kSlots = 16;
constexpr int kKVHeads = 4;
constexpr int kQHeads = 32;
constexpr int kGroup = kQHeads / kKVHeads;  // 8 query heads per kv head
constexpr int kHeadDim = 64;

constexpr int kMaxSegs = 4;                        // sequences per bin
constexpr int kMaxUnits = 256;                     // blocks per bin
constexpr int kHeaderInts = 8;                     // {segments, blocks, plan epoch, 0 x 5}
constexpr int kSegInts = 8;                        // {sequence, length, first block, blocks, first bin, part, parts, first slot}
constexpr int kRecordInts = kHeaderInts + kMaxSegs * kSegInts;
constexpr int kRowInts = kRecordInts + kMaxUnits;  // one plan row: the record, then the block ids
constexpr int kGroups = 8;                         // XCDs of an MI355X
constexpr int kTargetBins = 256;                   // CUs of an MI355X
constexpr int kMinBinBlocks = 8;                   // smaller workloads use fewer bins
constexpr int kSlotBytes = 2176;                   // partial: O (2 KiB, lane-major), (m, l) x 8, flag; 17 lines
constexpr int kFlagOffset = 2112;
constexpr int kMaxSpins = 100000;                  // bounded wait for a part's flag
constexpr int kWorkspaceHeader = PC_ATTN_WORKSPACE_HEADER_BYTES;  // the fault word, then reserved
constexpr uint32_t kEpochMask = (1u << 22) - 1;    // plan epochs occupy flag bits 9..30
static_assert(kWorkspaceHeader % 256 == 0, "partial slots keep the workspace's 256-byte alignment");

// A raised part flag: the plan's epoch in bits 9..30, the layer in bits 4..8 and the
// writer's XCD id + 1 in bits 0..3. A flag counts for a call only if its epoch and layer
// are the call's, so a flag left raised by an earlier call (a producer whose merge gave up
// waiting, or a plan without a merging row) is never taken for this call's partial: the
// merge keeps waiting until this call's producer overwrites it.
__device__ __forceinline__ int flag_key(int epoch, int layer) {
  return static_cast<int>(((static_cast<uint32_t>(epoch) & kEpochMask) << 9) | (static_cast<uint32_t>(layer) << 4));
}
__device__ __forceinline__ bool flag_of_call(int f, int key) { return (f & 0xF) != 0 && (f & ~0xF) == key; }

// Blocks holding `len` tokens, without the int32 overflow of len + 15.
__device__ __host__ __forceinline__ int blocks_of(int len) { return len / kSlots + (len % kSlots != 0); }

__device__ __forceinline__ int xcc_id() {
  int v;
  asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(v));
  return v & 0xff;
}

// LDS ordering inside one wave.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Workspace slot of part k of a cut sequence whose parts start at slot `first` (the plan
// numbers the parts of all cut sequences densely; the last part has no slot). `slots` is
// the workspace past its header.
__device__ __forceinline__ char* part_slot(char* slots, int first, int k, int h) {
  return slots + ((static_cast<int64_t>(first) + k) * kKVHeads + h) * kSlotBytes;
}

inline int check_attn_shape(int32_t batch, int32_t max_blocks) {
  using pc_internal::set_error;
  if (batch < 0 || batch > (1 << 20)) return set_error(PC_ERR_ARGUMENT, "batch %d out of range", batch);
  if (max_blocks < 1 || max_blocks > (1 << 16)) {
    return set_error(PC_ERR_ARGUMENT, "max_blocks %d out of range [1, 65536]", max_blocks);
  }
  return PC_OK;
}

// Bins of one group the planner may create for a batch of `batch` sequences of at most
// `max_blocks` blocks: the nominal cut (at most the whole target, or one bin per kMaxUnits
// blocks when that is more), plus one early close per kMaxSegs - 1 complete sequences (a bin
// closed at kMaxSegs segments holds at least that many), plus one.
inline int64_t group_bins_bound(int32_t batch, int32_t max_blocks) {
  const int64_t total = static_cast<int64_t>(batch) * max_blocks;
  const int64_t nominal = std::max<int64_t>(kTargetBins, (total + kMaxUnits - 1) / kMaxUnits);
  return nominal + 1 + (batch + kMaxSegs - 2) / (kMaxSegs - 1) + 1;
}

// Plan rows (workgroups) that always suffice for the shape.
inline int64_t plan_rows_bound(int32_t batch, int32_t max_blocks) {
  return static_cast<int64_t>(kGroups) * group_bins_bound(batch, max_blocks);
}

// `threads`: of a workgroup, which takes a row. A launch of 2^32 threads or more would be done modulo 2^32, without an error.
inline int check_plan_rows(int32_t num_records, int32_t batch, int32_t max_blocks, int threads) {
  using pc_internal::set_error;
  if (num_records < 0 || num_records > plan_rows_bound(batch, max_blocks)) {
    return set_error(PC_ERR_ARGUMENT, "num_records %d outside [0, pc_attn_plan_capacity]", num_records);
  }
  const int64_t most = ((int64_t{1} << 32) - 1) / threads / kGroups * kGroups;
  if (num_records > most) return set_error(PC_ERR_ARGUMENT, "num_records %d above %lld, a launch's", num_records, static_cast<long long>(most));
  return PC_OK;
}

// Partial slots that always suffice: one per bin at most (a bin ends at most one cut part
// that is not a sequence's last). The bins over all groups number at most the target plus
// one per kMaxUnits blocks plus rounding (kGroups x 1.5), plus the early closes.
inline int64_t slots_bound(int32_t batch, int32_t max_blocks) {
  const int64_t total = static_cast<int64_t>(batch) * max_blocks;
  return kTargetBins + (total + kMaxUnits - 1) / kMaxUnits + 2 * kGroups + (batch + kMaxSegs - 2) / (kMaxSegs - 1);
}

// The header (fault word), then the partial slots.
inline int64_t workspace_bytes_for(int64_t slots) { return kWorkspaceHeader + slots * kKVHeads * kSlotBytes; }

}  // namespace attn_plan

#endif  // PAGEDCORE_ATTN_PLAN_H
