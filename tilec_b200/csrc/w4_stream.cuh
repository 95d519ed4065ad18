// w4_stream.cuh -- the few-rows product with 4-bit weights on mma.sync: one row of 16-bit x on the
// integer path, up to 16 rows of 16-bit x and up to 8 of fp32 x on the 16-bit one.
//
// One token's product reads N * K / 2 bytes of codes and is bound by memory, if only the
// arithmetic keeps up: at 6.5 TB/s a quarter SM has about 180 cycles per 1 KB of codes (16
// rows x 128 k).  As 16-bit floats (multiply16: 0x4300 | code is 128 + code in bf16, 0x6400 |
// code is 1024 + code in fp16, minus 128 + zero; products are exact, sums fp32, the scale
// multiplies a group's sum) a code costs 1.4 instructions, most of them on the half-rate integer
// pipe.  fp32 x enters as three bf16 numbers of 8 bits each, which hold all of its 24 (w4_stage32):
// three columns of the product to a row of x.
// An 8-bit operand (multiply8) needs 3 for 8 codes, and m16n8k32 takes twice the k at the
// same rate, for the eight columns that one row of x then has:
//
//   * per 128-k block, x becomes pairs of whole numbers X 2^(e - 29) + Y 2^(e - 60), 2^e <= the
//     block's largest magnitude < 2^(e + 1), in four signed 8-bit digits each.  That is all of a
//     16-bit number down to 2^-53 (bf16; fp16: always) of the largest.  What they leave out of
//     smaller ones is kept in a list (W4Rest, normally empty) and added by itself: x enters exactly;
//   * each digit is one column of the tensor-core product, so sums over a group are exact
//     32-bit integers: sum code * digit - zero * sum digit;
//   * that times scale * the digit's power of two is added in fp32.
// (With X alone an fp32 element 2^-13 of its block's largest keeps 17 bits, which shows where the
// largest meets the zero point: 4e-6 off where an fp32 product is 2e-7.)
//
// The sums start at 0x4B400000 - zero * sum X: read as a float that is 1.5 * 2^23 + the sum
// (|sum| < 2^22), which saves the conversions.
//
// One CTA per SM, persistent, with 16 warps that share one copy of x.  A CTA takes an equal
// run of 16-row tiles, and its warps equal runs of their pieces (16 rows x 128 k): a warp's
// run is one run of memory too, streamed through a ring of its own in shared memory by bulk
// copies of four pieces each (two where x needs the room), so that 140 (70) KB are on their way
// to an SM at any time.  Where a
// tile is shared by several warps their sums meet in shared memory, in the order of K.
// Each CTA cuts, splits or copies x for itself, a slab of K at a time where it does not fit (one
// row: from K = 10368 or less on).
//
// Measured (graph replay), 28672 x 8192, one token (125 MB): 26.2 us, 4.8 TB/s; four digits
// instead of eight 25.4, but eight are what holds x, and the other four columns of the MMA would be
// idle.  On the way, with 27.8 as the best then: rows of codes with the group words apart 35 to 40 us
// (the words alone cost 6); 24 warps with copies of two pieces 30.5; 12 warps 30.3; CTAs of
// 128 rows, two waves of them for want of one slot, 40.  8 rows: 33.2 us (a grid of small CTAs
// with cp.async rings 48), 16 rows, x in three slabs: 50.4.  fp32: one row 32.3, 8 rows of 8192 x
// 8192 34.1 (in digits 28.4 and 34.4).
#pragma once

#include <cfloat>

#include "tc2_f16.cuh"
#include "w4.cuh"

namespace tilec {

constexpr int kW4StreamWarps = 16;
constexpr int kW4Digits = 8;      // columns of the one row of x
constexpr int kW4GroupTiles = 16; // row tiles whose sums a CTA holds at a time

// The digits of x in shared memory; zeros past K.
struct W4Digits {
  uint8_t* digits;   // [col][pitch], 128 bytes a block, [t][j][8]: 8 consecutive k in the order 0 4 1 5 2 6 3 7
  int64_t pitch;
  int* sums;         // [block][group][8]: minus the sum of a column's digits over a group
  float* scale;      // [block][8]: 2^(e - 60) * 256^digit for the lower four, 2^(e - 29) * 256^(digit - 4)
  int gpb;           // groups per block
  int* rest_count;   // elements of the slab that the digits do not hold in full ...
  struct W4Rest* rest;  // ... and by how much, kW4MaxRest at most
};

// An element of x beyond what its digits hold: its k, and the exact difference.
struct W4Rest {
  int k;
  float value;
};
constexpr int kW4MaxRest = 64;

struct W4StreamArgs {
  W4Args w;          // the weight, x, bias and out
  int row_tiles;
  int per_cta;       // blocks of K a CTA takes; a cluster's CTAs follow one another along K
  int slab;          // blocks of x in shared memory at a time
  int polling;       // the device's wait limit is shortened (w4_wait_on)
};

// XT: how x enters: 0 in digits (one 16-bit row), TILEC_DTYPE_F16 or _BF16 as it is, kW4Terms
// (fp32) in three bf16 terms.
constexpr int kW4Terms = 3;

template <int NT, int GPB, bool WIDE, int XT>
struct W4StreamCfg {
  static constexpr int kThreads = 32 * kW4StreamWarps;
  static constexpr int kPiece = w4_piece_bytes(GPB, WIDE);
  // Pieces a copy.  An SM's bulk copies start some 60 ns apart, so few large ones keep up with
  // HBM; with more columns, or 16-bit x, x needs the room (16-bit x, 3 rows: no faster with four).
  static constexpr int kRun = XT == 0 && NT == 1 && kPiece <= 1152 ? 4 : 2;
  static constexpr int kStage = kRun * kPiece;
  static constexpr int kStages = 2;
  static constexpr int kRingBytes = kW4StreamWarps * kStages * kStage;
  static constexpr bool kSummed = XT == 0 || XT == kW4Terms;  // several columns to a row of x
  static_assert(kW4GroupTiles * 16 * 8 * NT <= 32 * kThreads, "a bit per output of a thread");
  static_assert(!(XT == 0 && NT != 1) && !(XT == kW4Terms && NT != 1 && NT != 3), "columns of several to a row");
  static constexpr int kRows = XT == 0 ? 1 : kSummed && NT == 1 ? 2 : kSummed ? 8 : 8 * NT;  // rows of x
  static constexpr int kPart = kRows * 16;  // floats: the sums of a row tile, [row of x][16]
  // Chains of MMAs per group and column: one of eight dependent MMAs is what a warp would wait for
  // (28672 x 8192, 8 rows: 38.9 us, in two parts 34.8, in four 37.7); three tiles of columns are
  // three chains already.
  static constexpr int kChains = NT == 3 ? 1 : 2;
  static constexpr int kSumBytes = kW4GroupTiles * kPart * 4;
  static constexpr int kPartBytes = 2 * kW4StreamWarps * kPart * 4;
  static constexpr int kBarBytes = 1024;     // a barrier per warp and stage, rows' states, W4Rest, the abort flag
  static constexpr int kStatesAt = 256;      // w4_row_states of 16 rows, and whether they are wanted
  static constexpr int kRestAt = 512 - 16;   // two counts, then the entries
  static constexpr int kFixed = kRingBytes + kSumBytes + kPartBytes + kBarBytes;
  static_assert(kStage % 128 == 0 && kW4StreamWarps * kStages * 8 <= kStatesAt, "shared memory layout");
  static_assert(kStatesAt + 17 * 4 <= kRestAt, "shared memory layout");
  static_assert(kRestAt + 8 + kW4MaxRest * 8 <= kBarBytes - 8, "shared memory layout");
};
// Bytes of `slab` blocks of x: digits (16 bytes more a column: conflict-free reads), sums, scales.
__host__ __device__ inline int64_t w4_slab_bytes(int64_t slab, int gpb) {
  return kW4Digits * (slab * kW4Block + 16) + slab * kW4Digits * 4 * (gpb + 1);
}
// The same in 16-bit values (64 bytes more a row: conflict-free reads); fp32: three such rows.
__host__ __device__ inline int64_t w4_slab16_bytes(int64_t slab, int64_t rows) {
  return rows * (slab * (2 * kW4Block) + 64);
}

// Sixteen lanes (l = 0 .. 15) cut one 128-k block of the row x; all lanes of a warp call.
// `at`: where the block goes in d.
__device__ __forceinline__ void w4_cut(const W4Args& p, const W4Digits& d, bool live, int blk, int at, int l) {
  const int j = l >> 2, t = l & 3;
  const int k0 = blk * kW4Block + 8 * l;
  float v[8];
  const unsigned short* src = static_cast<const unsigned short*>(p.x) + k0;
  uint32_t w[4] = {0, 0, 0, 0};
  if (live && p.vec_x && k0 + 8 <= p.K) {
    const uint4 h = *reinterpret_cast<const uint4*>(src);
    w[0] = h.x; w[1] = h.y; w[2] = h.z; w[3] = h.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (live && k0 + i < p.K) w[i >> 1] |= uint32_t(src[i]) << (16 * (i & 1));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (p.dtype == 2) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  uint32_t top = 0;  // the largest magnitude, as bits: infinities and NaN come out on top
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  // Powers of two as bits.  2^-60 and below share one step, so that all of them are normal numbers.
  const int e = max(static_cast<int>(top >> 23) - 127, -60);
  auto pow2 = [](int n) { return __uint_as_float(static_cast<uint32_t>(127 + n) << 23); };
  // x = X 2^(e - 29) + Y 2^(e - 60), |X|, |Y| <= 2^30, and what neither holds.
  uint32_t x_hi[8], x_lo[8];  // with 0x80 in every byte: bytes, less 0x80 each, are the digits
  auto cut = [&](uint32_t (&y)[8], float up, float down) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int whole = __float2int_rn(v[i] * up);
      y[i] = static_cast<uint32_t>(whole) + 0x80808080u;
      v[i] = fmaf(-__int2float_rn(whole), down, v[i]);  // exact: few bits of x are left below a step
    }
  };
  cut(x_hi, pow2(29 - e), pow2(e - 29));
  cut(x_lo, pow2(60 - e), pow2(e - 60));
  bool rest = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) rest |= v[i] != 0.f;
  if (rest && top < 0x7F800000u) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float value = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) value = c == i ? v[c] : value;
      if (value == 0.f) continue;
      const int n = atomicAdd(d.rest_count, 1);
      if (n < kW4MaxRest) d.rest[n] = W4Rest{k0 + i, value};
    }
  }
  // A block with anything not finite makes its sums NaN, and the outputs are then computed one by
  // one (w4_output).
  const bool finite = top < 0x7F800000u;
#pragma unroll
  for (int col = 0; col < kW4Digits; ++col) {
    const int part = col & 3;
    const uint32_t(&y)[8] = col < 4 ? x_lo : x_hi;
    const uint32_t sel = part | (4 + part) << 4;
    auto gather = [&](int a, int b, int c, int e) {
      return __byte_perm(__byte_perm(y[a], y[b], sel), __byte_perm(y[c], y[e], sel), 0x5410) ^ 0x80808080u;
    };
    const uint32_t d0 = gather(0, 4, 1, 5), d1 = gather(2, 6, 3, 7);
    int sum = __dp4a(static_cast<int>(d0), 0x01010101, __dp4a(static_cast<int>(d1), 0x01010101, 0));
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    int other = __shfl_xor_sync(0xffffffffu, sum, 4);
    if (d.gpb <= 2) sum += other;
    other = __shfl_xor_sync(0xffffffffu, sum, 8);
    if (d.gpb == 1) sum += other;
    if (!live) continue;
    *reinterpret_cast<uint2*>(d.digits + col * d.pitch + at * kW4Block + t * 32 + j * 8) = make_uint2(d0, d1);
    if (t == 0 && j % (4 / d.gpb) == 0) d.sums[(at * d.gpb + j / (4 / d.gpb)) * kW4Digits + col] = -sum;
    if (l == 0)
      d.scale[at * kW4Digits + col] = finite ? pow2(e - (col < 4 ? 60 : 29) + 8 * part) : __int_as_float(0x7fc00000);
  }
}

__device__ __forceinline__ float w4_weight(const W4Args& p, int gpb, int n, int k) {
  const int wb = w4_word_bytes(gpb, p.wide), b = k / kW4Block, kk = k % kW4Block;
  const uint8_t* piece = p.data + (int64_t(n >> 4) * p.blocks + b) * w4_piece_bytes(gpb, p.wide);
  const uint32_t code = reinterpret_cast<const uint32_t*>(piece + 16 * wb + (n & 15) * 64)[(kk >> 3 & 3) * 4 + (kk >> 5)];
  const uint32_t* w = reinterpret_cast<const uint32_t*>(piece + (n & 15) * wb) + (kk * gpb / kW4Block) * (p.wide ? 2 : 1);
  const float s = p.wide ? __uint_as_float(w[1]) : w4_scale16(w[0], p.scale_bf16);
  return (float((code >> (4 * (kk >> 1 & 3) + 16 * (kk & 1))) & 15u) - float(w[0] & 15u)) * s;
}

// What x's digits left out, in order of k: the sum over `n` entries for one output.
__device__ __noinline__ float w4_rest(const W4Args& p, int gpb, int row, const W4Rest* list, int n) {
  float v = 0.f;
  for (int i = 0; i < n; ++i) v += list[i].value * w4_weight(p, gpb, row, list[i].k);
  return v;
}

// One output from its definition, in fp32 and k order: where the digits'
// sums are not finite because x is not, or where codes times an x of 2^117 or more are past fp32's
// range before the scale brings them back.  Slow: some 0.5 to 5 ms for a weight's outputs.
__device__ __noinline__ float w4_output(const W4Args& p, int gpb, int n, int m) {
  float v = 0.f;
  for (int k = 0; k < p.K; ++k) {
    v += load_as_float(p.x, m * p.ldx + k, p.dtype) * w4_weight(p, gpb, n, k);
    if (v != v) break;  // it stays NaN
  }
  return v;
}

// Whether rows of x hold infinities (bit 0 of states[m]) or NaN (bit 1).  All threads of a CTA call;
// asked only where an output is not finite.
__device__ __noinline__ void w4_row_states(const W4Args& p, int* states) {
  const bool wide = p.dtype == TILEC_DTYPE_F32;
  const uint32_t top = wide ? 0x7F800000u : p.dtype == TILEC_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  for (int m = 0; m < p.M; ++m) {
    int state = 0;
    for (int k = threadIdx.x; k < p.K; k += 32 * kW4StreamWarps) {
      const int64_t at = m * p.ldx + k;
      const uint32_t bits = wide ? static_cast<const uint32_t*>(p.x)[at] & 0x7FFFFFFFu
                                 : static_cast<const unsigned short*>(p.x)[at] & 0x7FFFu;
      if (bits >= top) state |= bits == top ? 1 : 2;
    }
    if (state != 0) atomicOr(&states[m], state);
  }
  __syncthreads();
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Shared memory by its 32-bit address: one register and an immediate where generic pointers
// cost two registers and their arithmetic.
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t (&w)[WORDS], uint32_t a) {
  if constexpr (WORDS == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
  } else if constexpr (WORDS == 2) {
    const uint2 v = lds64(a);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 v = lds128(a + 4 * i);
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
}

// 16-bit rows of x, blocks s0 .. s0 + n, to shared memory: [row][pitch], zeros past K.
__device__ __forceinline__ void w4_stage16(const W4Args& p, uint8_t* xs, int pitch, int s0, int n) {
  const int per_row = n * (kW4Block / 8);
  for (int i = threadIdx.x; i < p.M * per_row; i += 32 * kW4StreamWarps) {
    const int m = i / per_row, c = i - m * per_row, k = s0 * kW4Block + 8 * c;
    const unsigned short* s = static_cast<const unsigned short*>(p.x) + m * p.ldx + k;
    uint8_t* dst = xs + m * pitch + 16 * c;
    if (p.vec_x && k + 8 <= p.K) {
      cp_async_16(dst, s, 16);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < p.K) w[j >> 1] |= uint32_t(s[j]) << (16 * (j & 1));
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  cp_async_commit();
  cp_async_wait<0>();
}

// fp32 rows of x, blocks s0 .. s0 + n, as three bf16 numbers each: x = high + middle + low, 8 bits
// of its 24 each, cut off and not rounded (nothing overflows, nothing is lost down to 2^-133).
// [term][row][pitch], zeros past K.  Infinities and NaN are their own high term.
__device__ __forceinline__ void w4_stage32(const W4Args& p, uint8_t* xs, int pitch, int s0, int n) {
  const int per_row = n * (kW4Block / 8);
  for (int i = threadIdx.x; i < p.M * per_row; i += 32 * kW4StreamWarps) {
    const int m = i / per_row, c = i - m * per_row, k = s0 * kW4Block + 8 * c;
    const float* s = static_cast<const float*>(p.x) + m * p.ldx + k;
    float v[8];
    if (p.vec_x && k + 8 <= p.K) {
      const float4 a = reinterpret_cast<const float4*>(s)[0], b = reinterpret_cast<const float4*>(s)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < p.K ? s[j] : 0.f;
    }
#pragma unroll
    for (int term = 0; term < kW4Terms; ++term) {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = __float_as_uint(v[j]);
        h[j] = bits & 0xFFFF0000u;
        if ((bits & 0x7F800000u) == 0x7F800000u) {
          if ((bits & 0x007FFFFFu) != 0) h[j] = 0x7FC00000u;  // a NaN whose high half may say infinity
          v[j] = 0.f;
        } else {
          v[j] -= __uint_as_float(h[j]);
        }
      }
      *reinterpret_cast<uint4*>(xs + (term * p.M + m) * pitch + 16 * c) =
          make_uint4(__byte_perm(h[0], h[1], 0x7632), __byte_perm(h[2], h[3], 0x7632),
                     __byte_perm(h[4], h[5], 0x7632), __byte_perm(h[6], h[7], 0x7632));
    }
  }
}

// What a warp does when a copy has not landed after one try (mbar_wait's loop, out of line).
// `polling`: the device's limit is shortened (failure tests).  The suspending form of the test
// sleeps for longer than a copy takes, so with it no limit below that would ever run out.
__device__ __noinline__ bool w4_wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag, bool polling) {
  const unsigned long long t0 = global_ns(), limit = wait_limit();
  for (;;) {
    if (polling) {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(bar), "r"(parity)
          : "memory");
      if (done) return true;
    } else if (mbar_try<false>(bar, parity, kHintStage)) {
      return true;
    }
    if (*abort_flag) return false;
    if (global_ns() - t0 > limit) {
      *abort_flag = 1;
      record_status(TILEC_DEV_TIMEOUT);
      return false;
    }
  }
}

// SC: type of the scales (TILEC_DTYPE_*); where x is not in digits (XT != 0) 0, or 1 for either 16-bit type.
// Grid: x = CTAs (clusters of `splits`, whose CTAs share their row tiles and split K).
template <int NT, int GPB, int SC, int XT>
__global__ void __launch_bounds__(32 * kW4StreamWarps, 1) w4_stream_kernel(const __grid_constant__ W4StreamArgs a) {
  constexpr bool WIDE = SC == 0;
  using Cfg = W4StreamCfg<NT, GPB, WIDE, XT>;
  constexpr int WB = w4_word_bytes(GPB, WIDE), T = Cfg::kThreads, S = Cfg::kStages, W = kW4StreamWarps;
  constexpr bool BF = XT == TILEC_DTYPE_BF16 || XT == kW4Terms;  // bf16 operands (where x is not in digits)
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const W4Args& p = a.w;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = w4_smem + warp * (S * Cfg::kStage);
  float* tile_sums = reinterpret_cast<float*>(w4_smem + Cfg::kRingBytes);                  // [tile of the group][kPart]
  float* parts = reinterpret_cast<float*>(w4_smem + Cfg::kRingBytes + Cfg::kSumBytes);     // [warp][first, last][kPart]
  uint64_t* bars = reinterpret_cast<uint64_t*>(w4_smem + Cfg::kFixed - Cfg::kBarBytes) + warp * S;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(w4_smem + Cfg::kFixed - 8);
  const int pitch = XT == 0 ? a.slab * kW4Block + 16 : a.slab * (2 * kW4Block) + 64;
  W4Digits d;                                      // the slab of x
  d.digits = w4_smem + Cfg::kFixed;
  d.pitch = pitch;
  d.sums = reinterpret_cast<int*>(d.digits + p.cols * pitch);
  d.scale = reinterpret_cast<float*>(d.sums + a.slab * GPB * 8);
  d.gpb = GPB;
  int* rest_counts = reinterpret_cast<int*>(w4_smem + Cfg::kFixed - Cfg::kBarBytes + Cfg::kRestAt);  // of slabs in turn
  d.rest = reinterpret_cast<W4Rest*>(rest_counts + 2);
  int* row_states = reinterpret_cast<int*>(w4_smem + Cfg::kFixed - Cfg::kBarBytes + Cfg::kStatesAt);
  volatile int* again_flag = row_states + 16;  // some output was not finite
  const int g = lane >> 2, t = lane & 3;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = static_cast<int>(blockIdx.x) / p.splits, clusters = static_cast<int>(gridDim.x) / p.splits;
  const int b_begin = min(p.blocks, rank * a.per_cta), b_end = min(p.blocks, b_begin + a.per_cta);
  const int tile_begin = static_cast<int>(int64_t(a.row_tiles) * cluster / clusters);
  const int tile_end = static_cast<int>(int64_t(a.row_tiles) * (cluster + 1) / clusters);
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
    if (warp == 0) *abort_flag = rest_counts[0] = rest_counts[1] = 0;
    fence_barrier_init();
  }
  if (threadIdx.x <= 16) row_states[threadIdx.x] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  float total[NT][4];
  // 32-bit shared addresses; columns past the last one repeat it, their sums are never read.
  const uint32_t ring_at = smem_u32(ring), lane_codes = 16 * WB + lane * 16, lane_words = g * WB;
  uint32_t x_col[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    // Three terms to a row: columns 4 * row + term (the fourth is not read), or a tile of columns per term.
    const int row = XT != kW4Terms ? min(8 * i + g, p.cols - 1)
                    : NT == 1      ? min(g & 3, 2) * p.M + min(g >> 2, p.M - 1)
                                   : i * p.M + min(g, p.M - 1);
    x_col[i] = smem_u32(d.digits) + row * pitch + (XT == 0 ? 32 : 16) * t;
  }
  uint32_t magic = 0;  // in a register: the logic instruction takes one immediate
  if constexpr (XT != 0) asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF ? 0x43004300u : 0x64006400u));
  const uint32_t sums_at = smem_u32(d.sums) + 8 * t, scale_at = smem_u32(d.scale) + 8 * t;

  auto multiply16 = [&](uint32_t piece, int blk) {
    const uint4 qa = lds128(piece + lane_codes), qb = lds128(piece + lane_codes + 512);
    uint32_t wa[WB / 4], wb[WB / 4];
    lds_words(wa, piece + lane_words);
    lds_words(wb, piece + lane_words + 8 * WB);
    constexpr int CH = Cfg::kChains;
    float acc[NT][CH][4], sa = 0.f, sb = 0.f;
    uint32_t za = 0, zb = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int kSteps = 4 / GPB;  // words of codes per group
      if (j % kSteps == 0) {
        const int k = j / kSteps;
        const uint32_t ga = wa[WIDE ? 2 * k : k], gb = wb[WIDE ? 2 * k : k];
        if constexpr (WIDE) {
          sa = __uint_as_float(wa[2 * k + 1]);
          sb = __uint_as_float(wb[2 * k + 1]);
        } else {
          sa = w4_scale16(ga, p.scale_bf16);
          sb = w4_scale16(gb, p.scale_bf16);
        }
        za = magic | __byte_perm(ga, 0, 0x1010);
        zb = magic | __byte_perm(gb, 0, 0x1010);
      }
      const uint32_t ca = j == 0 ? qa.x : j == 1 ? qa.y : j == 2 ? qa.z : qa.w;
      const uint32_t cb = j == 0 ? qb.x : j == 1 ? qb.y : j == 2 ? qb.z : qb.w;
      uint32_t u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = w4_pair<BF>(ca, i, magic, za);
        v[i] = w4_pair<BF>(cb, i, magic, zb);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 xv = lds128(x_col[i] + blk * (2 * kW4Block) + 64 * j);
        if (j % kSteps == 0)
          mma_16816_zero<BF>(acc[i][0], u[0], v[0], u[1], v[1], xv.x, xv.y);
        else
          mma_16816<BF>(acc[i][0], u[0], v[0], u[1], v[1], xv.x, xv.y);
        if (j % kSteps == 0 && CH == 2)
          mma_16816_zero<BF>(acc[i][CH - 1], u[2], v[2], u[3], v[3], xv.z, xv.w);
        else
          mma_16816<BF>(acc[i][CH - 1], u[2], v[2], u[3], v[3], xv.z, xv.w);
      }
      if ((j + 1) % kSteps == 0) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            total[i][c] = fmaf(CH == 2 ? acc[i][0][c] + acc[i][CH - 1][c] : acc[i][0][c], c < 2 ? sa : sb, total[i][c]);
        }
      }
    }
  };
  auto multiply8 = [&](uint32_t piece, int blk) {
    const uint4 qa = lds128(piece + lane_codes), qb = lds128(piece + lane_codes + 512);
    uint32_t wa[WB / 4], wb[WB / 4];
    lds_words(wa, piece + lane_words);
    lds_words(wb, piece + lane_words + 8 * WB);
    uint4 x[NT][2];
    uint2 xs[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      x[i][0] = lds128(x_col[i] + blk * kW4Block);
      x[i][1] = lds128(x_col[i] + blk * kW4Block + 16);
      xs[i] = lds64(scale_at + blk * 32);
    }
    int acc[NT][4];
    float sa = 0.f, sb = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int kSteps = 4 / GPB;  // words of codes per group
      if (j % kSteps == 0) {
        const int k = j / kSteps;
        const uint32_t ga = wa[WIDE ? 2 * k : k], gb = wb[WIDE ? 2 * k : k];
        const int za = static_cast<int>(ga & 15u), zb = static_cast<int>(gb & 15u);
        if constexpr (WIDE) {
          sa = __uint_as_float(wa[2 * k + 1]);
          sb = __uint_as_float(wb[2 * k + 1]);
        } else {
          sa = w4_scale16(ga, SC == 2);
          sb = w4_scale16(gb, SC == 2);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint2 sx = lds64(sums_at + (blk * GPB + k) * 32);
          acc[i][0] = 0x4B400000 + za * static_cast<int>(sx.x);
          acc[i][1] = 0x4B400000 + za * static_cast<int>(sx.y);
          acc[i][2] = 0x4B400000 + zb * static_cast<int>(sx.x);
          acc[i][3] = 0x4B400000 + zb * static_cast<int>(sx.y);
        }
      }
      const uint32_t ca = j == 0 ? qa.x : j == 1 ? qa.y : j == 2 ? qa.z : qa.w;
      const uint32_t cb = j == 0 ? qb.x : j == 1 ? qb.y : j == 2 ? qb.z : qb.w;
      const uint32_t a0 = ca & 0x0F0F0F0Fu, a2 = (ca >> 4) & 0x0F0F0F0Fu;
      const uint32_t a1 = cb & 0x0F0F0F0Fu, a3 = (cb >> 4) & 0x0F0F0F0Fu;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 xv = x[i][j >> 1];
        const uint32_t b_lo = j & 1 ? xv.z : xv.x, b_hi = j & 1 ? xv.w : xv.y;
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+r"(acc[i][0]), "+r"(acc[i][1]), "+r"(acc[i][2]), "+r"(acc[i][3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b_lo), "r"(b_hi));
      }
      if ((j + 1) % kSteps == 0) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float x0 = __uint_as_float(xs[i].x), x1 = __uint_as_float(xs[i].y);
          total[i][0] = fmaf(__int_as_float(acc[i][0]) - 12582912.f, sa * x0, total[i][0]);
          total[i][1] = fmaf(__int_as_float(acc[i][1]) - 12582912.f, sa * x1, total[i][1]);
          total[i][2] = fmaf(__int_as_float(acc[i][2]) - 12582912.f, sb * x0, total[i][2]);
          total[i][3] = fmaf(__int_as_float(acc[i][3]) - 12582912.f, sb * x1, total[i][3]);
        }
      }
    }
  };

  auto multiply = [&](uint32_t piece, int blk) {  // `blk`: the piece's block within the slab
    if constexpr (XT == 0) multiply8(piece, blk);
    else multiply16(piece, blk);
  };

  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  int turn = 1, n_rest = 0;  // digits: the slab's count of W4Rest, and how many
  bool have_states = false;
  const bool whole_x = b_end - b_begin <= a.slab;
  for (int group = tile_begin; group < tile_end; group += kW4GroupTiles) {
    const int ntiles = min(kW4GroupTiles, tile_end - group);
    for (int s0 = b_begin; s0 == b_begin || s0 < b_end; s0 += a.slab) {
      const int n = max(0, min(a.slab, b_end - s0));  // blocks of K in work
      // This warp's run of the slab's pieces, tile by tile.
      const int pieces = ntiles * n, share = (pieces + W - 1) / W;
      const int first = min(pieces, warp * share), last = min(pieces, first + share);
      const int first_tile = n > 0 ? first / n : 0, first_blk = first - first_tile * n;
      // Up to kRun pieces of one tile follow one another in memory and go out in one copy.
      // Once this warp gave up it sends for nothing more: its barriers are no longer kept up.
      const bool in_step = ok;
      int f_left = ok ? last - first : 0, f_blk = first_blk, fill = stage;
      const uint8_t* f_src =
          p.data + (static_cast<int64_t>(group + first_tile) * p.blocks + s0 + f_blk) * Cfg::kPiece;
      const int64_t skip = static_cast<int64_t>(p.blocks - n) * Cfg::kPiece;  // from a tile's slab to the next one's
      auto fetch = [&]() {
        if (f_left <= 0) return;
        const int run = min(Cfg::kRun, min(f_left, n - f_blk));
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars[fill], run * Cfg::kPiece);
          bulk_load(ring + fill * Cfg::kStage, f_src, run * Cfg::kPiece, &bars[fill]);
        }
        fill = fill == S - 1 ? 0 : fill + 1;
        f_left -= run;
        f_blk += run;
        f_src += run * Cfg::kPiece;
        if (f_blk == n) {
          f_blk = 0;
          f_src += skip;
        }
      };
#pragma unroll
      for (int i = 0; i < S; ++i) fetch();
      const bool stage_x = !whole_x || (group == tile_begin && s0 == b_begin);
      if (stage_x) {
        turn ^= 1;
        d.rest_count = rest_counts + turn;
        if constexpr (XT == kW4Terms) {
          w4_stage32(p, d.digits, pitch, s0, n);
        } else if constexpr (XT != 0) {
          w4_stage16(p, d.digits, pitch, s0, n);
        } else {
          for (int base = 0; base < n; base += T / 16) {
            const int at = base + (threadIdx.x >> 4);
            w4_cut(p, d, at < n, s0 + at, at, threadIdx.x & 15);
          }
        }
      }
      if (s0 == b_begin)
        for (int i = threadIdx.x; i < ntiles * Cfg::kPart; i += T) tile_sums[i] = 0.f;
      __syncthreads();
      if constexpr (XT == 0) {
        if (stage_x) {
          n_rest = rest_counts[turn];
          if (threadIdx.x == 0) rest_counts[turn ^ 1] = 0;  // last read before the slab's first barrier
          if (n_rest > 1 && n_rest <= kW4MaxRest) {  // in order of k, whoever came first
            W4Rest mine = {};
            int rank = 0;
            if (static_cast<int>(threadIdx.x) < n_rest) {
              mine = d.rest[threadIdx.x];
              for (int i = 0; i < n_rest; ++i) rank += d.rest[i].k < mine.k;
            }
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < n_rest) d.rest[rank] = mine;
            __syncthreads();
          }
        }
      }

      // A row tile's sums are complete, or as far as this warp goes.
      auto leave = [&](int tile, bool whole, int which) {
        float* dst = whole ? tile_sums + tile * Cfg::kPart : parts + (2 * warp + which) * Cfg::kPart;
        if constexpr (Cfg::kSummed && NT == 1) {
          // A row of x: its digits in all four lanes t, or its terms in two of them (three of four columns).
          const bool both = XT == 0 || (t & 1) == 0;
          float v0 = total[0][0] + (both ? total[0][1] : 0.f), v1 = total[0][2] + (both ? total[0][3] : 0.f);
          v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
          v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
          if constexpr (XT == 0) {
            v0 += __shfl_xor_sync(0xffffffffu, v0, 2);
            v1 += __shfl_xor_sync(0xffffffffu, v1, 2);
          }
          if (XT == 0 ? t == 0 : (t & 1) == 0) {
            float* r = dst + (t >> 1) * 16 + g;
            r[0] = whole ? r[0] + v0 : v0;
            r[8] = whole ? r[8] + v1 : v1;
          }
        } else {
#pragma unroll
          for (int i = 0; i < (Cfg::kSummed ? 1 : NT); ++i) {
            float* r = dst + (8 * i + 2 * t) * 16 + g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float* at = r + (j & 1) * 16 + (j >> 1) * 8;
              float v = total[i][j];
              if constexpr (Cfg::kSummed) v = (total[2][j] + total[1][j]) + total[0][j];
              *at = whole ? *at + v : v;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) total[i][0] = total[i][1] = total[i][2] = total[i][3] = 0.f;
      };
#pragma unroll
      for (int i = 0; i < NT; ++i) total[i][0] = total[i][1] = total[i][2] = total[i][3] = 0.f;
      int tile = first_tile, blk = first_blk;
      bool from_start = blk == 0;   // this warp has the tile's first block
      for (int at = first; at < last && ok;) {
        const uint32_t bar = smem_u32(&bars[stage]);
        ok = __all_sync(0xffffffffu, (!a.polling && mbar_try<false>(bar, phase, kHintStage)) ||
                                         w4_wait_on(bar, phase, abort_flag, a.polling));
        if (!ok) break;
        const uint32_t piece = ring_at + stage * Cfg::kStage;
        const int run = min(Cfg::kRun, min(last - at, n - blk));
#pragma unroll
        for (int i = 0; i < Cfg::kRun; ++i)
          if (i < run) multiply(piece + i * Cfg::kPiece, blk + i);
        __syncwarp();  // every lane has read the stage
        fetch();
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
        at += run;
        blk += run;
        if (blk == n) {
          leave(tile, from_start, tile == first_tile ? 0 : 1);
          ++tile;
          blk = 0;
          from_start = true;
        }
      }
      if (ok && first < last && blk > 0) leave(tile, false, tile == first_tile ? 0 : 1);
      if (!ok) {  // gave up, here or earlier: let what is on its way land, and leave NaN
        if (in_step) {
          const int on_way = fill == stage ? S : (fill - stage + S) % S;  // one at least: the one waited for
          for (int i = 0; i < on_way; ++i) {
            const int at = (stage + i) % S;
            mbar_drain(&bars[at], at >= stage ? phase : phase ^ 1);
          }
        }
        for (int i = lane; i < 2 * Cfg::kPart; i += 32) parts[2 * warp * Cfg::kPart + i] = __int_as_float(0x7fc00000);
        for (int k = first; k < last; k = (k / n + 1) * n)
          for (int i = lane; i < Cfg::kPart; i += 32) tile_sums[k / n * Cfg::kPart + i] = __int_as_float(0x7fc00000);
      }
      __syncthreads();
      // Tiles that several warps share: the first of them adds the parts, in the order of K.
      if (first < last) {
        auto gather = [&](int tl) {
          const int lo = tl * n, hi = lo + n;
          if (first > lo || last >= hi) return;  // an earlier warp leads, or this one had it whole
          for (int i = lane; i < Cfg::kPart; i += 32) {
            float v = tile_sums[tl * Cfg::kPart + i];
            for (int w = warp; w < W && w * share < hi; ++w)  // w's first tile, unless it starts before
              v += parts[(2 * w + (w * share >= lo ? 0 : 1)) * Cfg::kPart + i];
            tile_sums[tl * Cfg::kPart + i] = v;
          }
        };
        gather(first_tile);
        const int last_tile = (last - 1) / n;
        if (last_tile != first_tile) gather(last_tile);
      }
      __syncthreads();
      if constexpr (XT == 0) {
        if (n_rest > 0) {  // rare; more than the list holds: the outputs are computed one by one
          for (int i = threadIdx.x; i < ntiles * 16; i += T)
            tile_sums[i] += n_rest > kW4MaxRest ? __int_as_float(0x7fc00000)
                                                : w4_rest(p, GPB, group * 16 + i, d.rest, n_rest);
          __syncthreads();
        }
      }
    }

    // Outputs of the group's tiles, from all CTAs' sums of a cluster.
    if (p.splits > 1) cluster_sync();
    const int count = ntiles * 16 * p.M;
    auto put = [&](int i, float v) {
      const int row = group * 16 + (i >> 4) / p.M * 16 + (i & 15), m = (i >> 4) % p.M;
      if (p.bias != nullptr) v += load_as_float(p.bias, row, p.dtype);
      store_from_float(p.out, int64_t(m) * p.ldo + row, p.dtype, v);
    };
    uint32_t again = 0;  // this thread's outputs that are not finite, one bit each
    int turn_out = 0;
    for (int i = rank * T + threadIdx.x; i < count; i += p.splits * T, ++turn_out) {
      const int r = i & 15, m = (i >> 4) % p.M, tl = (i >> 4) / p.M, at = tl * Cfg::kPart + m * 16 + r;
      if ((group + tl) * 16 + r >= p.N) continue;
      float v = 0.f;
      if (p.splits == 1) {
        v = tile_sums[at];
      } else {
        const uint32_t addr = smem_u32(tile_sums + at);
        for (int c = 0; c < p.splits; ++c) {
          float u;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(mapa_shared(addr, c)) : "memory");
          v += u;
        }
      }
      if (XT != TILEC_DTYPE_F16 && !(fabsf(v) <= FLT_MAX)) again |= 1u << turn_out;
      put(i, v);
    }
    if (again) *again_flag = 1;
    if (p.splits > 1) cluster_sync();  // every CTA's sums have been read
    else __syncthreads();
    // Sums that are not finite though x is have left fp32's range (fp16 cannot), or were given up;
    // an x in digits that is not finite has none.
    if constexpr (XT != TILEC_DTYPE_F16) {
      if (*again_flag) {
        if (!have_states) w4_row_states(p, row_states);
        have_states = true;
        for (; again; again &= again - 1) {
          const int i = rank * T + threadIdx.x + (__ffs(again) - 1) * p.splits * T, m = (i >> 4) % p.M;
          if (XT == 0 ? (row_states[m] & 2) == 0 : row_states[m] == 0)
            put(i, w4_output(p, GPB, group * 16 + (i >> 4) / p.M * 16 + (i & 15), m));
        }
      }
    }
  }
}

}  // namespace tilec
