// 8-bit projection of a decode step's rows: Y = X W^T with W e4m3 [n][k] and X e4m3 or fp16 [m][k],
// both with a power of two per row and block of 128 columns (fp8_device.h). It takes the place of
// torch.nn.functional.linear on fp16 weights (reference src/pagedcore/dense.py:91-104 via
// src/pagedcore/decoder.py:156-199).
//
//   Y[i][j] = sum over blocks b of 2^(sx[i][b] + sw[j][b]) * (sum over l in b of x[i][l] w[j][l])
//
// The weight is the stream: n k bytes from HBM, half of what the fp16 form reads. One workgroup
// computes 16 MT rows of X times 16 NT rows of W; its waves take runs of the split's blocks of 128 columns,
// so every byte of the tile is fetched by exactly one wave, through a ring
// of D slots of its own (LDS DMA, whole 128-byte lines), with no barrier in the loop. The waves' sums
// are added in wave order at the end. SwiGLU of 1 row (11264 x 2048) 6.6 us, of which a launch is 1.9: 4.9 TB/s behind it, a
// large copy's rate; of 24 rows 7.9-8.1 us, where the X that every workgroup fetches again counts too.
//
// fp16 outputs run on the 8-bit matrix instruction of 128 columns, which takes the powers of two itself.
// It adds eight products at a time aligned to the largest and drops what lies below 2^-13 of it: measured 1.5e-5 of the
// result's norm on normal data, 3e-5 where one column in a hundred is ten times as large. The rounding to fp16 that
// follows is 2.1e-4 (together 2.10e-4 against 2.07e-4). The fp32 partial sums
// run on the fp16 instruction, the operands widened from e4m3 in registers (exact; 5e-8), since what
// adds them decides what they are rounded to. An fp16 X is rounded to 8 bits in registers, with the values and
// scales of pc_quantize_fp8, so that a decode step needs no launch for it.

#include "fp8_gemm.h"

#include <iterator>

namespace fp8_gemm {
namespace {

using namespace fp8_device;
using namespace rope_device;
using gemm_device::float4_t;
using gemm_device::half4_t;
using gemm_device::half8_t;
using gemm_device::lds_offset;
using gemm_device::lds_ptr;
using gemm_device::raise_lds_limit;
using gemm_device::wait_vm;
using pc_internal::check_launch;

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef short short2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

// The words of a 16-byte LDS chunk.
__device__ __forceinline__ uint4_t lds_words(uint32_t addr) {
  return *reinterpret_cast<const __attribute__((address_space(3))) uint4_t*>(static_cast<uintptr_t>(addr));
}
__device__ __forceinline__ uint32_t lds_word(uint32_t addr) {
  return *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(static_cast<uintptr_t>(addr));
}

// Eight e4m3 as fp16, exactly.
__device__ __forceinline__ half8_t widen(uint32_t a, uint32_t b) {
  const half2_t p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
  const half2_t q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
  const half2_t r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
  const half2_t s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
  return half8_t{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// Eight fp16 divided by `scale`, a power of two, rounded to e4m3 (the conversion divides by its scale
// operand exactly before it rounds, and turns infinities and NaN into NaN).
__device__ __forceinline__ uint2_t round_fp8(half8_t v, float scale) {
  short2_t a{}, b{};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, half2_t{v[0], v[1]}, scale, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, half2_t{v[2], v[3]}, scale, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, half2_t{v[4], v[5]}, scale, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, half2_t{v[6], v[7]}, scale, true);
  return uint2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// What X holds past its columns.
__device__ const uint4 zeros[1] = {};

// The larger of two pairs of fp16 magnitudes, as bits (so that infinities and NaN come out on top).
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t a, uint32_t b) {
  typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}

template <int MT, int NT, int WAVES, int D, bool HALFX>
struct Shape {
  static constexpr int XB = MT * (HALFX ? 4096 : 2048);  // X part of a unit: 16 MT rows of 128 columns
  static constexpr int WB = NT * 2048;
  static constexpr int UB = XB + WB;
  static constexpr int PER = UB / 1024;                  // DMA instructions per unit
  static constexpr int SB = HALFX ? 256 : 512;           // four blocks' scales: W's rows, then X's
  static constexpr int WAVE = D * UB + 2 * SB;
  static constexpr int RING = WAVES * WAVE;
  static constexpr int SUMS = WAVES * MT * NT * 1024;
  static constexpr int LDS = RING > SUMS ? RING : SUMS;
  static_assert(LDS <= 160 * 1024, "ring and accumulator exchange fit the CU's LDS");
  static_assert((D - 1) * PER < 64 && D >= 1 && D <= 4, "vmcnt counts the later units");
  static_assert(NT <= 4 && MT <= 4, "one scale word per lane");
};

// The arguments that only the end of the kernel reads; those before it are preloaded into SGPRs at wave
// launch (no kernel-argument round trip before the first DMA).
struct Rest {
  void* out;
  const int64_t* slots;
  RopeOut rope;
};

template <int MT, int NT, int WAVES, int D, bool HALFX, Form E>
__global__ __launch_bounds__(64 * WAVES) void fp8_stream_kernel(const void* x, const uint8_t* w, const uint8_t* x_scales,
                                                                const uint8_t* w_scales, int m, int n, int k,
                                                                int splits_mtiles, const int64_t* positions, Rest rest) {
  using S = Shape<MT, NT, WAVES, D, HALFX>;
  constexpr int kRowsX = 16 * MT;
  constexpr int kCols = paired(E) ? 8 * NT : 16 * NT;  // output columns per tile (pairs of them)
  constexpr bool kExact = E == kPartials;
  constexpr int kXSize = HALFX ? 2 : 1;                // bytes per element of X
  constexpr int kXBytes = S::XB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r16 = lane & 15, g = lane >> 4;
  const int limit = paired(E) ? n / 2 : n;
  const int tiles = (limit + kCols - 1) / kCols;
  const int splits = splits_mtiles >> 16, mtiles = splits_mtiles & 65535;
  // Workgroups of one W tile (one per X tile) are 8 apart, on one XCD: W comes from HBM once.
  int id = blockIdx.x, mtile = 0;
  if (mtiles > 1) {
    const int q = id >> 3;
    mtile = q % mtiles;
    id = (q / mtiles) * 8 + (id & 7);
  }
  const int tile = id % tiles, split = id / tiles;
  if (split >= splits) return;  // the grid is rounded up to 8 tiles
  const int blocks = (k + kBlock - 1) / kBlock;
  const int first = static_cast<int>(static_cast<int64_t>(split) * blocks / splits);
  const int end = static_cast<int>(static_cast<int64_t>(split + 1) * blocks / splits);
  // This wave's blocks: a run of them, so that four in a row share the words of their scales.
  const int begin = first + wave * (end - first) / WAVES;
  const int mine = first + (wave + 1) * (end - first) / WAVES - begin;

  // Row r of the tile's W part, relative to its first; rows past the matrix repeat its last row.
  const int last = limit - 1 - kCols * tile, last_x = m - 1 - kRowsX * mtile;
  auto w_row = [&](int r) {
    if constexpr (E == kSwiGLU) return r < kCols ? min(r, last) : limit + min(r - kCols, last);
    else if constexpr (E == kRope) return pair_row(kCols * tile) + (r < kCols ? r : kHalfDim + r - kCols);
    else return min(r, last);
  };
  // DMA of 1 KiB: eight rows of 128 bytes (lane L takes row L / 8 and the chunk stored at position
  // L % 8: chunk c of row r at c ^ (r & 7)), or four fp16 rows of 256 (position c ^ (r & 15)).
  const int row8 = lane >> 3;
  const int chunk = 16 * ((lane & 7) ^ row8);
  uint32_t xoff[kXBytes / 1024], woff[2 * NT];
  int xchunk[kXBytes / 1024];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i) woff[i] = static_cast<uint32_t>(w_row(8 * i + row8)) * static_cast<uint32_t>(k);
#pragma unroll
  for (int i = 0; i < kXBytes / 1024; ++i) {
    const int r = HALFX ? 4 * i + (lane >> 4) : 8 * i + row8;
    xoff[i] = static_cast<uint32_t>(min(r, last_x)) * static_cast<uint32_t>(k * kXSize);
    xchunk[i] = HALFX ? 16 * ((lane & 15) ^ (r & 15)) : chunk;
  }
  const char* const xbase = static_cast<const char*>(x) + static_cast<int64_t>(kRowsX) * mtile * k * kXSize;
  const uint8_t* const wbase = w + (E == kRope ? 0 : static_cast<int64_t>(kCols) * tile * k);
  const int stride = scale_stride(k);
  const uint8_t* const xscale = HALFX ? nullptr : x_scales + (static_cast<int64_t>(kRowsX) * mtile + min(min(lane, kRowsX - 1), last_x)) * stride;
  const uint8_t* const wscale = w_scales + ((E == kRope ? 0 : static_cast<int64_t>(kCols) * tile) + w_row(min(lane, 16 * NT - 1))) * stride;
  // RoPE: thread e ends with quad e % Q of row e / Q of the tile (one each at most). Its position
  // and slot are loaded before the stream's first unit and the table values behind it, so that
  // the stream hides both round trips (loads return in order: an older one in flight only
  // makes the waits below longer).
  constexpr int T = MT * NT, Q = kCols / 4;  // Q: groups of four output columns
  static_assert(E != kRope || (kHalfDim % kCols == 0 && Q * kRowsX <= 64 * WAVES), "one quad of one head per thread");
  int64_t position = 0, slot_of = 0;
  if constexpr (E == kRope) {
    const int row = min(kRowsX * mtile + static_cast<int>(threadIdx.x) / Q, m - 1);
    position = positions[row];
    slot_of = (rest.slots != nullptr ? rest.slots : positions)[row];
  }
  char* const ring = smem + wave * S::WAVE;
  char* const scale_ring = ring + D * S::UB;
  constexpr int kScaleBytes = S::SB;
  auto issue = [&](char* slot, int t) {
    const int b = begin + t;
    const int left = k - kBlock * b;  // columns of this block and later ones
    const uint8_t* const wblock = wbase + static_cast<int64_t>(kBlock) * b;
    const char* const xblock = xbase + static_cast<int64_t>(kBlock * kXSize) * b;
    // Chunks past the columns, in the last block alone: X's are zeros, W's chunk 0 of their row in place.
    const int wc = chunk < left ? chunk : 0;
    asm volatile("" ::: "memory");
    // The scales of blocks b & ~3 .. + 3, with the first of them that this wave takes (ahead of its data: the
    // waits count the data's instructions, and two more in flight only make one of them longer).
    if (t == 0 || (b & 3) == 0) {
      char* const words = scale_ring + ((b >> 2) & 1) * kScaleBytes;
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(wscale + (b & ~3)), lds_ptr(words), 4, 0, 0);
      if constexpr (!HALFX) {
        __builtin_amdgcn_global_load_lds(static_cast<const void*>(xscale + (b & ~3)), lds_ptr(words + 256), 4, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(wblock + (woff[i] + wc)), lds_ptr(slot + kXBytes + i * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < kXBytes / 1024; ++i) {
      const char* const src = xchunk[i] < left * kXSize ? xblock + (xoff[i] + xchunk[i]) : reinterpret_cast<const char*>(zeros);
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(src), lds_ptr(slot + i * 1024), 16, 0, 0);
    }
    asm volatile("" ::: "memory");
  };

  float4_t acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  const uint32_t ring0 = lds_offset(ring);
  // 32 fp16 of a row's block in this lane, 128 in the four lanes of the row: rounded, and the scale.
  auto round_row = [&](uint32_t base, uint4_t (&eight)[2], int& scale) {
    half8_t v[4];
    uint32_t most = 0;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int c = 8 * (f >> 1) + 2 * g + (f & 1);
      const uint4_t words = lds_words(base + r16 * 256 + ((c ^ r16) * 16));
      v[f] = __builtin_bit_cast(half8_t, words);
#pragma unroll
      for (int e = 0; e < 4; ++e) most = max_magnitudes(most, words[e] & 0x7fff7fffu);
    }
    auto widest = [](uint32_t bits) {  // over the row's lanes; non-negative floats and fp16 compare as their bits do
      const auto p = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
      const uint32_t half = max(p[0], p[1]);
      const auto q = __builtin_amdgcn_permlane16_swap(half, half, false, false);
      return max(q[0], q[1]);
    };
    most = widest(max(most & 0xffffu, most >> 16));
    float largest = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(most)));
    if (__builtin_amdgcn_ballot_w64(most >= 0x7c00u)) {  // an infinity or NaN in some row: the largest of the others
      float finite = 0.0f;
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int e = 0; e < 8; ++e) finite = fmaxf(finite, finite_magnitude(static_cast<float>(v[f][e])));
      largest = __uint_as_float(widest(__float_as_uint(finite)));
    }
    scale = scale_of(largest);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint2_t a = round_fp8(v[2 * p], power_of(scale)), b = round_fp8(v[2 * p + 1], power_of(scale));
      eight[p] = uint4_t{a[0], a[1], b[0], b[1]};
    }
  };
  // The block t of this wave in slot d. Lane (r16, g) holds columns 16 g .. + 15 and 64 + 16 g .. + 15 of
  // row r16 of each 16 rows.
  auto unit = [&](int d, int t) {
    const int b = begin + t;
    const uint32_t scales = ring0 + D * S::UB + ((b >> 2) & 1) * S::SB;
    const int shift = 8 * (b & 3);
    const uint32_t base = ring0 + d * S::UB;
    uint4_t x8[MT][2];
    int xs[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if constexpr (HALFX) {
        round_row(base + j * 4096, x8[j], xs[j]);
      } else {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          x8[j][p] = lds_words(base + j * 2048 + r16 * 128 + (((4 * p + g) ^ (r16 & 7)) * 16));
        }
        xs[j] = (lds_word(scales + 256 + (16 * j + r16) * 4) >> shift) & 255;
      }
    }
    if constexpr (kExact) {
      half8_t xf[MT][4];
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int f = 0; f < 4; ++f) xf[j][f] = widen(x8[j][f >> 1][2 * (f & 1)], x8[j][f >> 1][2 * (f & 1) + 1]);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        half8_t wf[4];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint4_t words = lds_words(base + S::XB + i * 2048 + r16 * 128 + (((4 * p + g) ^ (r16 & 7)) * 16));
          wf[2 * p] = widen(words[0], words[1]);
          wf[2 * p + 1] = widen(words[2], words[3]);
        }
        const uint4_t words = lds_words(scales + (16 * i + 4 * g) * 4);
        float4_t sum[MT];
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int j = 0; j < MT; ++j)
            sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[f], xf[j][f], f ? sum[j] : float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float sw = power_of((words[e] >> shift) & 255);
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j][e] = fmaf(sum[j][e] * power_of(xs[j]), sw, acc[i][j][e]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        int8v_t wf;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint4_t words = lds_words(base + S::XB + i * 2048 + r16 * 128 + (((4 * p + g) ^ (r16 & 7)) * 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) wf[4 * p + e] = static_cast<int>(words[e]);
        }
        const int ws = (lds_word(scales + (16 * i + r16) * 4) >> shift) & 255;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          int8v_t xf;
#pragma unroll
          for (int e = 0; e < 8; ++e) xf[e] = static_cast<int>(x8[j][e >> 2][e & 3]);
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[i][j], 0, 0, 0, ws, 0, xs[j]);
        }
      }
    }
  };

#pragma unroll
  for (int t = 0; t < D; ++t) {
    if (t < mine) issue(ring + t * S::UB, t);
  }
  [[maybe_unused]] RopeRow rope{};
  [[maybe_unused]] half4_t cs{}, sn{};
  if constexpr (E == kRope) {
    rope = rope_row(rest.rope, position, slot_of, rest.slots != nullptr);
    const _Float16* table = rope.table + (kCols * tile + 4 * (static_cast<int>(threadIdx.x) % Q)) % kHalfDim;
    cs = *reinterpret_cast<const half4_t*>(table);
    sn = *reinterpret_cast<const half4_t*>(table + kHalfDim);
  }
  // Unit t in slot t % D: its DMA has landed once at most the later units' are outstanding.
  for (int t = 0; t < mine; ++t) {
    const int later = min(D - 1, mine - 1 - t);
    if (D > 3 && later == 3) wait_vm<(D > 3 ? 3 : 1) * S::PER>();
    else if (D > 2 && later == 2) wait_vm<(D > 2 ? 2 : 1) * S::PER>();
    else if (later == 1) wait_vm<S::PER>();
    else wait_vm<0>();
    const int d = t % D;
    unit(d, t);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its reads are done before the slot is refilled
    if (t + D < mine) issue(ring + d * S::UB, t + D);
  }

  // Sums to LDS (over the rings, once every wave is done with its own), then added in wave order:
  // acc[i][j] of lane (r16, g) holds X row 16 j + r16, W rows 16 i + 4 g .. + 3.
  __syncthreads();
  float4_t* sums = reinterpret_cast<float4_t*>(smem);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[(wave * T + i * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < Q * kRowsX; e += 64 * WAVES) {
    const int q = e % Q, r = e / Q;
    const int row = kRowsX * mtile + r, col = kCols * tile + 4 * q;
    auto total = [&](int quad) {
      const float4_t* p = sums + ((quad >> 2) * MT + (r >> 4)) * 64 + 16 * (quad & 3) + (r & 15);
      float4_t v = p[0];
#pragma unroll
      for (int u = 1; u < WAVES; ++u) v += p[u * T * 64];
      return v;
    };
    if (row >= m || col >= limit) continue;
    const float4_t v = total(q);
    if constexpr (E == kPartials) {
      float* y = static_cast<float*>(rest.out) + (static_cast<int64_t>(split) * m + row) * n + col;
      *reinterpret_cast<float4_t*>(y) = v;
    } else {
      half4_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = static_cast<_Float16>(v[i]);
      if constexpr (E == kHalf) {
        *reinterpret_cast<half4_t*>(static_cast<_Float16*>(rest.out) + static_cast<int64_t>(row) * n + col) = o;
      } else {
        const float4_t u = total(Q + q);
        if constexpr (E == kSwiGLU) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = static_cast<_Float16>(silu_mul(v[i], u[i]));
          *reinterpret_cast<half4_t*>(static_cast<_Float16*>(rest.out) + static_cast<int64_t>(row) * limit + col) = o;
        } else {
          half4_t high;
#pragma unroll
          for (int i = 0; i < 4; ++i) high[i] = static_cast<_Float16>(u[i]);
          store_pairs(rest.rope, rope, row, col, o, high, cs, sn);
        }
      }
    }
  }
}

template <int MT, int NT, int WAVES, int D, bool HALFX, Form E>
int launch(const Args& a, hipStream_t s) {
  using S = Shape<MT, NT, WAVES, D, HALFX>;
  constexpr int cols = paired(E) ? 8 * NT : 16 * NT;
  auto kernel = fp8_stream_kernel<MT, NT, WAVES, D, HALFX, E>;
  static std::atomic<uint64_t> raised{0};
  if (int rc = raise_lds_limit(reinterpret_cast<const void*>(kernel), S::LDS, raised)) return rc;
  const int tiles = ((paired(E) ? a.n / 2 : a.n) + cols - 1) / cols;
  const int mtiles = (a.m + 16 * MT - 1) / (16 * MT);
  int64_t grid = static_cast<int64_t>(tiles) * a.splits;
  if (mtiles > 1) grid = (grid + 7) / 8 * 8 * mtiles;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * WAVES), S::LDS, s, a.x, a.w, a.x_scales,
                     a.w_scales, a.m, a.n, a.k, a.splits * 65536 + mtiles, a.positions, Rest{a.out, a.slots, a.rope});
  return check_launch("fp8_stream_gemm");
}

// The instances, in the four cases of what X is and what the products run on. The constants are fitted to
// the times of every instance at 19000 calls (m 1 to 2048, n 256 to 11264, k 256 to 5632, 1 to 8 splits, every form,
// weights from HBM): the instance taken, of these and the tiles, is 1.5 % off the fastest of all that were measured on
// average, more than 20 % off at 2 % of the calls (1.7 times at worst, where a second round has few workgroups).
// Rings of two units, three where a 16 x 16 tile leaves the LDS for them, and of one where that lets a second workgroup
// onto the CU, which hides more than a second unit: fp32 partial sums of 8-bit rows a seventh faster over
// the calls above, of fp16 rows, which fill twice the LDS, a seventh (down of 128 rows at 4 splits 14.4 -> 12.8 us, 13.2 with
// outputs that are not in the caches). On the
// 8-bit instruction a second unit is as good or better (32 x 48 tiles of one unit, for SwiGLU of 17 to 32 rows: 8.7 us, the 32 x 32
// tiles of two 7.7 to 8.2). Where a workgroup per CU is all there is, more in flight in it is faster: a second unit, or eight
// waves (down of 16 rows at 4 splits 6.8 us / 5.8).
struct Instance {
  int mt, nt, waves, units;
  Cost cost;
};
constexpr Instance kEight[] = {  // e4m3 X on the 8-bit instruction
    {1, 1, 4, 3, {2.07f, 0.17f, 0.22f, 0.08f}}, {1, 2, 4, 2, {2.14f, 0.01f, 0.33f, 0.12f}},
    {2, 2, 4, 2, {1.98f, 0.33f, 0.41f, 0.12f}}, {3, 2, 4, 2, {0.92f, 1.54f, 0.55f, 0.12f}},
    {4, 2, 4, 2, {0.91f, 1.68f, 0.64f, 0.13f}}, {4, 3, 4, 2, {0.92f, 2.18f, 0.78f, 0.13f}},
    {4, 4, 4, 2, {0.96f, 2.24f, 0.94f, 0.14f}},
};
constexpr Instance kEightExact[] = {  // e4m3 X widened: fp32 partial sums
    {1, 2, 4, 2, {2.17f, 0.1f, 0.47f, 0.09f}}, {2, 2, 4, 1, {2.47f, 0.0f, 0.6f, 0.11f}}, {4, 2, 4, 1, {2.83f, 0.02f, 0.96f, 0.14f}},
};
constexpr Instance kHalfX[] = {  // fp16 X rounded, on the 8-bit instruction
    {1, 1, 4, 3, {2.15f, 0.19f, 0.5f, 0.03f}},  {1, 2, 4, 2, {2.18f, 0.09f, 0.55f, 0.1f}}, {2, 4, 4, 2, {0.88f, 1.81f, 1.27f, 0.15f}},
    {1, 2, 8, 2, {0.82f, 1.35f, 0.92f, 0.13f}}, {2, 2, 8, 1, {0.96f, 1.43f, 1.4f, 0.2f}},
};
constexpr Instance kHalfXExact[] = {
    {1, 1, 4, 3, {1.95f, 0.35f, 0.55f, 0.04f}}, {1, 2, 4, 1, {2.56f, 0.0f, 0.58f, 0.11f}},  {1, 2, 4, 2, {2.11f, 0.26f, 0.68f, 0.08f}},
    {1, 2, 8, 2, {1.04f, 1.3f, 1.17f, 0.11f}},  {2, 2, 8, 1, {1.07f, 1.46f, 1.71f, 0.19f}}, {2, 4, 4, 1, {2.79f, 0.0f, 1.7f, 0.12f}},
};

// Whether an instance can end with the rotation, as the kernel asserts, and adds in the order of the others that can.
constexpr bool rotates(const Instance& i) {
  return i.waves == 4 && kHalfDim % (8 * i.nt) == 0 && 2 * i.nt * 16 * i.mt <= 64 * i.waves;
}

template <int N>
Choice fastest(const Args& a, Form form, const Instance (&instances)[N]) {
  Choice best{-1, INFINITY};
  for (int i = 0; i < N; ++i) {
    const Instance& t = instances[i];
    if (i > 0 && 16 * (t.mt - 1) >= a.m) continue;  // a second X tile without rows
    if (qkv_product(a, form) && !rotates(t)) continue;
    const int cols = paired(form) ? 8 * t.nt : 16 * t.nt, width = paired(form) ? a.n / 2 : a.n;
    const int blocks = (a.k + kBlock - 1) / kBlock;
    const int64_t workgroups =
        static_cast<int64_t>((width + cols - 1) / cols) * a.splits * ((a.m + 16 * t.mt - 1) / (16 * t.mt));
    const float time = estimate(t.cost, workgroups, ((blocks + a.splits - 1) / a.splits + t.waves - 1) / t.waves, a);
    if (time < best.time) best = Choice{i, time};
  }
  return best;
}

template <Form E, bool HALFX, const auto& INSTANCES, size_t I = 0>
int launch_index(const Args& a, size_t index, hipStream_t s) {
  if constexpr (I == sizeof(INSTANCES) / sizeof(Instance)) {
    return pc_internal::set_error(PC_ERR_ARGUMENT, "no kernel instance %d", static_cast<int>(index));
  } else {
    constexpr Instance t = INSTANCES[I];
    if constexpr (E != kRope || rotates(t)) {
      if (index == I) return launch<t.mt, t.nt, t.waves, t.units, HALFX, E>(a, s);
    }
    return launch_index<E, HALFX, INSTANCES, I + 1>(a, index, s);
  }
}

template <Form E>
int launch_form(const Args& a, int index, hipStream_t s) {
  if constexpr (E == kPartials) {
    return a.x_scales ? launch_index<E, false, kEightExact>(a, index, s) : launch_index<E, true, kHalfXExact>(a, index, s);
  } else {
    return a.x_scales ? launch_index<E, false, kEight>(a, index, s) : launch_index<E, true, kHalfX>(a, index, s);
  }
}

}  // namespace

Choice choose_stream(const Args& a, Form form, bool half_x) {
  if (form == kPartials) return half_x ? fastest(a, form, kHalfXExact) : fastest(a, form, kEightExact);
  return half_x ? fastest(a, form, kHalfX) : fastest(a, form, kEight);
}

int stream_kernels(Form form, bool half_x) {
  return static_cast<int>(form == kPartials ? (half_x ? std::size(kHalfXExact) : std::size(kEightExact))
                                            : (half_x ? std::size(kHalfX) : std::size(kEight)));
}

int launch_stream(const Args& a, Form form, int index, hipStream_t s) {
  switch (form) {
    case kPartials: return launch_form<kPartials>(a, index, s);
    case kHalf: return launch_form<kHalf>(a, index, s);
    case kSwiGLU: return launch_form<kSwiGLU>(a, index, s);
    default: return launch_form<kRope>(a, index, s);
  }
}

}  // namespace fp8_gemm
