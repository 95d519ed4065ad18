// w4.cuh -- products with 4-bit weights: y[m, n] = sum_k x[m, k] * (code[n, k] - zero) * scale,
// scale and zero per group of consecutive k.
//
// Layout of the weight (made once by the caller): 16 rows x 128 k at a time, [row tile][block
// of 128 k], each such piece in one run of memory: the 16 rows' group words, then 64 bytes of
// codes a row.  A warp that walks along K reads one stream (one token, 28672 x 8192: 27.8 us;
// rows of codes with the words apart: 35 at best).
//   Codes of a row and block: word 4t + j (t, j = 0..3) holds k = 32j + 8t + 0..7, the even ones
//   of these in nibbles 0..3 and the odd ones in nibbles 4..7.  So
//     * lane t of the four lanes that share a row takes its words 4t .. 4t+3, 16 bytes;
//     * word j of all four lanes covers k = 32j .. 32j+31, i.e. one group even when groups are
//       32 long;
//     * (word >> 4i) & 0x000F000F is the pair k = 2i, 2i+1, next to each other as x is.
//   Group words: per group of the block (four of 32, two of 64, or one) a 32-bit word, zero |
//   scale << 16 (16-bit scales), or two, zero and the fp32 scale.  Groups longer than 128 have
//   theirs in every block.
//
// Up to some tens of rows of x the product streams the codes once (K/2 bytes a row of W).
// At full bandwidth an SM has under three lane-instructions per weight, too few to convert
// and multiply each weight on the FMA pipe, so the sums run on mma.sync: 16 rows of W against
// 8 columns at a time.  (tcgen05 would need the converted weights to pass through shared
// memory first; with so few columns its rate is not what bounds this.)  The fewest rows take
// the integer form (w4_stream.cuh); here, for 11 to 32 rows of 16-bit x, a code becomes a
// 16-bit float exactly: 0x4300 | code is 128 + code in bf16 (0x6400 | code is 1024 + code in
// fp16), minus (128 + zero).  Products are exact, sums fp32; the scale multiplies a group's
// fp32 sum.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tilec {

constexpr int kW4Warps = 8;
constexpr int kW4Block = 128;  // k per 64-byte block of codes

struct W4Args {
  const uint8_t* data;     // [row tiles][blocks][piece]
  int wide;                // fp32 scales: (zero, scale) pairs
  int scale_bf16;          // 16-bit scales: bf16 (else fp16)
  int N, K, blocks;
  const void* x;           // [M][ldx] of type dtype
  int64_t ldx;
  int dtype;               // TILEC_DTYPE_* of x, bias and out
  int M, cols;             // cols: M, or M times the digits of w4_stream_kernel
  int vec_x;               // 16-byte loads of x allowed (16-bit types)
  void* out;               // [M][ldo]
  int64_t ldo;
  const void* bias;        // [N] or nullptr
  int tiles;               // work tiles of w4_mma_kernel
  int splits;              // CTAs of a cluster that share a row tile's K
  int row_warps;           // warps of a CTA along rows (the others share its K)
  int slab;                // 128-k blocks of x in shared memory at a time
};

// Bytes of a piece (16 rows x 128 k): its group words, then its codes.
__host__ __device__ constexpr int w4_word_bytes(int gpb, bool wide) { return gpb * (wide ? 8 : 4); }  // of a row
__host__ __device__ constexpr int w4_piece_bytes(int gpb, bool wide) { return 16 * w4_word_bytes(gpb, wide) + 1024; }

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dt) {
  if (dt == 0) return static_cast<const float*>(p)[i];
  return load_16(p, i, dt == 2);
}
__device__ __forceinline__ void store_from_float(void* p, int64_t i, int dt, float v) {
  if (dt == 0)
    static_cast<float*>(p)[i] = v;
  else if (dt == 1)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float w4_scale16(uint32_t word, bool bf16) {
  return bf16 ? __uint_as_float(word & 0xFFFF0000u) : __half2float(__ushort_as_half(static_cast<unsigned short>(word >> 16)));
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The pair of codes i of a word, minus the zero point (zm = the magic number | zero, twice).
// The and-or is one three-input logic instruction; left to the compiler it became two, and
// the integer pipe is what this kernel's arithmetic runs into first.
template <bool BF16>
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, int i, uint32_t magic, uint32_t zm) {
  uint32_t v, r;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(magic));
  if constexpr (BF16)
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zm));
  else
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zm));
  return r;
}

// c = A B without an accumulator to clear first.
template <bool BF16>
__device__ __forceinline__ void mma_16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// `BYTES` bytes (4, 8 or a multiple of 16) to shared memory.
template <int BYTES>
__device__ __forceinline__ void cp_async_bytes(uint8_t* dst, const uint8_t* src) {
  if constexpr (BYTES == 4) {
    cp_async_4(dst, src, 4);
  } else if constexpr (BYTES == 8) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < BYTES; i += 16)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + i)), "l"(src + i) : "memory");
  }
}

// Columns of x in shared memory: [col][pitch] 16-bit values, k0 .. k0 + n (n a multiple of
// 128), zeros past K.
__device__ __forceinline__ void w4_stage_x(const W4Args& p, unsigned short* xs, int pitch, int k0, int n) {
  const int per_row = n / 8;
  for (int i = threadIdx.x; i < p.M * per_row; i += 32 * kW4Warps) {
    const int m = i / per_row, kk = (i - m * per_row) * 8, k = k0 + kk;
    const unsigned short* s = static_cast<const unsigned short*>(p.x) + m * p.ldx + k;
    uint4 h = make_uint4(0, 0, 0, 0);
    if (p.vec_x && k + 8 <= p.K) {
      h = *reinterpret_cast<const uint4*>(s);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < p.K) w[j >> 1] |= uint32_t(s[j]) << (16 * (j & 1));
      h = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(xs + m * pitch + kk) = h;
  }
}

// A warp owns 16 * MT rows of W; `row_warps` warps of a CTA lie along rows and the others
// take its 128-k blocks in turn, so that neighbours read neighbouring 64 bytes of a row; a
// cluster's CTAs split K once more.  Sums meet in shared memory, then over the cluster, in a
// fixed order.  CTAs are persistent over row tiles.  Codes and group words come through a ring
// of cp.async copies in which every thread reads only what it copied itself: no barrier, and
// kStages - 1 blocks of every warp are always on their way (each 1 KB x MT), across row tiles
// too, which is what keeps HBM busy; registers hold only the block in work.  x is staged for
// `slab` blocks at a time (once, if that is all of the CTA's K) and shared by its warps.
// GPB: scale groups per 128-k block (4, 2, or 1 for longer groups).  WIDE: fp32 scales.
// Grid: x = resident clusters of `splits` CTAs (at most one per row tile).
template <int MT, int GPB, bool WIDE>
struct W4Cfg {
  static constexpr int kRows = 2 * MT;  // rows per lane
  static constexpr int kThreads = 32 * kW4Warps;
  static constexpr int kWordBytes = GPB * (WIDE ? 8 : 4);  // of a row and block
  static constexpr int kStages = MT == 1 ? 5 : (kWordBytes > 16 ? 3 : 4);
  static constexpr int kCodeStage = kRows * 16 * kThreads;
  static constexpr int kWordStage = kRows * kWordBytes * kThreads;
  static constexpr int kRingBytes = kStages * (kCodeStage + kWordStage);
  static constexpr int kPerSm = MT == 1 ? 3 : 2;  // CTAs the registers allow on an SM
};

template <bool BF16, int NT, int MT, int GPB, bool WIDE>
__global__ void __launch_bounds__(32 * kW4Warps, W4Cfg<MT, GPB, WIDE>::kPerSm) w4_mma_kernel(const __grid_constant__ W4Args p) {
  using Cfg = W4Cfg<MT, GPB, WIDE>;
  constexpr int S = Cfg::kStages, R = Cfg::kRows, COLS = 8 * NT, WB = Cfg::kWordBytes;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int k_warps = kW4Warps / p.row_warps;
  const int row_warp = warp % p.row_warps, k_warp = warp / p.row_warps;
  const int tile_rows = 16 * MT * p.row_warps;
  const int clusters = static_cast<int>(gridDim.x) / p.splits;
  const int per_cta = (p.blocks + p.splits - 1) / p.splits;
  const int b_begin = min(p.blocks, rank * per_cta), b_end = min(p.blocks, b_begin + per_cta);
  uint8_t* code_ring = w4_smem + threadIdx.x * 16;                         // [stage][row][thread]
  uint8_t* word_ring = w4_smem + S * Cfg::kCodeStage + threadIdx.x * WB;   // [stage][row][thread]
  float* red = reinterpret_cast<float*>(w4_smem + Cfg::kRingBytes);        // [k_warp][row][col]
  unsigned short* xs = reinterpret_cast<unsigned short*>(red + kW4Warps * 16 * MT * COLS);
  const int pitch = p.slab * kW4Block + 32;  // + 64 bytes: the 8 lanes of a quarter read 8 different 16-byte banks
  pdl_wait();
  pdl_launch_dependents();

  // The fetching side runs ahead of the computing side, with its own tile, block and pointers.
  constexpr int PIECE = w4_piece_bytes(GPB, WIDE);
  const int row_tiles = (p.N + 15) / 16;
  int f_tile = static_cast<int>(blockIdx.x) / p.splits - clusters, f_b = b_end;
  const uint8_t* f_ptr[MT];
  auto fetch = [&](int slot) {  // the next block of this warp into ring slot `slot`
    if (f_b >= b_end) {
      f_tile += clusters;
      f_b = b_begin + k_warp;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int64_t rt = min((f_tile * p.row_warps + row_warp) * MT + m, row_tiles - 1);
        f_ptr[m] = p.data + (rt * p.blocks + f_b) * PIECE;
      }
    }
    if (f_tile < p.tiles && f_b < b_end) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint8_t* piece = f_ptr[i >> 1];
        cp_async_16(code_ring + slot * Cfg::kCodeStage + i * (16 * Cfg::kThreads),
                    piece + 16 * WB + (i & 1) * 512 + lane * 16, 16);
        cp_async_bytes<WB>(word_ring + slot * Cfg::kWordStage + i * (WB * Cfg::kThreads),
                           piece + (g + 8 * (i & 1)) * WB);
      }
    }
    cp_async_commit();
    f_b += k_warps;
#pragma unroll
    for (int m = 0; m < MT; ++m) f_ptr[m] += static_cast<int64_t>(k_warps) * PIECE;
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(i);

  uint32_t magic;  // in a register: the logic instruction takes one immediate
  asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300u : 0x64006400u));
  // Columns past the last one repeat it; their sums are never read.
  const unsigned short* xcol[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) xcol[i] = xs + min(8 * i + g, p.cols - 1) * pitch + 8 * t;
  const bool whole_x = b_end - b_begin <= p.slab;
  int slot = 0, fill = S - 1;
  bool staged = false;

  for (int tile = static_cast<int>(blockIdx.x) / p.splits; tile < p.tiles; tile += clusters) {
    float total[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) total[m][i][j] = 0.f;
    int b = b_begin + k_warp;
    for (int s0 = b_begin; s0 < b_end; s0 += p.slab) {
      const int s_end = min(b_end, s0 + p.slab);
      if (!staged) {
        __syncthreads();
        w4_stage_x(p, xs, pitch, s0 * kW4Block, (s_end - s0) * kW4Block);
        __syncthreads();
        staged = whole_x;
      }
      for (; b < s_end; b += k_warps) {
        fetch(fill);
        fill = fill == S - 1 ? 0 : fill + 1;
        cp_async_wait<S - 1>();
        uint4 q[R];
        uint32_t w[R][WB / 4];
#pragma unroll
        for (int i = 0; i < R; ++i) {
          q[i] = *reinterpret_cast<const uint4*>(code_ring + slot * Cfg::kCodeStage + i * (16 * Cfg::kThreads));
          const uint32_t* ws =
              reinterpret_cast<const uint32_t*>(word_ring + slot * Cfg::kWordStage + i * (WB * Cfg::kThreads));
#pragma unroll
          for (int k = 0; k < WB / 4; ++k) w[i][k] = ws[k];
        }
        slot = slot == S - 1 ? 0 : slot + 1;
        const unsigned short* xb[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) xb[i] = xcol[i] + (b - s0) * kW4Block;
        float acc[MT][NT][4], sc[R];
        uint32_t zm[R];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          constexpr int kSteps = 4 / GPB;  // words of codes per group
          if (j % kSteps == 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
              const int k = j / kSteps;
              if constexpr (WIDE)
                sc[i] = __uint_as_float(w[i][2 * k + 1]);
              else
                sc[i] = w4_scale16(w[i][k], p.scale_bf16);
              zm[i] = magic | __byte_perm(w[i][WIDE ? 2 * k : k], 0, 0x1010);
            }
          }
          uint4 xv[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) xv[i] = *reinterpret_cast<const uint4*>(xb[i] + 32 * j);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint4 qa = q[2 * m], qb = q[2 * m + 1];
            const uint32_t wa = j == 0 ? qa.x : j == 1 ? qa.y : j == 2 ? qa.z : qa.w;
            const uint32_t wb = j == 0 ? qb.x : j == 1 ? qb.y : j == 2 ? qb.z : qb.w;
            uint32_t a[4], c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              a[i] = w4_pair<BF16>(wa, i, magic, zm[2 * m]);
              c[i] = w4_pair<BF16>(wb, i, magic, zm[2 * m + 1]);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              if (j % kSteps == 0)
                mma_16816_zero<BF16>(acc[m][i], a[0], c[0], a[1], c[1], xv[i].x, xv[i].y);
              else
                mma_16816<BF16>(acc[m][i], a[0], c[0], a[1], c[1], xv[i].x, xv[i].y);
              mma_16816<BF16>(acc[m][i], a[2], c[2], a[3], c[3], xv[i].z, xv[i].w);
            }
            if ((j + 1) % kSteps == 0) {
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                total[m][i][0] = fmaf(acc[m][i][0], sc[2 * m], total[m][i][0]);
                total[m][i][1] = fmaf(acc[m][i][1], sc[2 * m], total[m][i][1]);
                total[m][i][2] = fmaf(acc[m][i][2], sc[2 * m + 1], total[m][i][2]);
                total[m][i][3] = fmaf(acc[m][i][3], sc[2 * m + 1], total[m][i][3]);
              }
            }
          }
        }
      }
    }
    // Sums of the tile: over the K warps, then over the cluster.
    const int n0 = tile * tile_rows, plane = tile_rows * COLS;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float* d = red + k_warp * plane + (16 * MT * row_warp + 16 * m + g) * COLS + 8 * i + 2 * t;
        *reinterpret_cast<float2*>(d) = make_float2(total[m][i][0], total[m][i][1]);
        *reinterpret_cast<float2*>(d + 8 * COLS) = make_float2(total[m][i][2], total[m][i][3]);
      }
    __syncthreads();
    auto finish = [&](int r, int m, auto sum_at) {
      const int n = n0 + r;
      if (n >= p.N) return;
      float v = sum_at(r * COLS + m);
      if (p.bias != nullptr) v += load_as_float(p.bias, n, p.dtype);
      store_from_float(p.out, int64_t(m) * p.ldo + n, p.dtype, v);
    };
    auto over_k_warps = [&](int i) {
      float v = red[i];
      for (int w = 1; w < k_warps; ++w) v += red[w * plane + i];
      return v;
    };
    if (p.splits == 1) {
      for (int i = threadIdx.x; i < tile_rows * p.M; i += Cfg::kThreads) finish(i % tile_rows, i / tile_rows, over_k_warps);
      __syncthreads();  // the sums have been read: the next tile may overwrite them
    } else {
      if (k_warps > 1) {
        for (int i = threadIdx.x; i < plane; i += Cfg::kThreads) red[i] = over_k_warps(i);  // red[i] is this thread's
      }
      cluster_sync();
      // Each CTA finishes its share of the rows from all CTAs' sums.
      const int share = (tile_rows + p.splits - 1) / p.splits;
      const int r0 = rank * share, rows = min(share, tile_rows - r0);
      auto over_cluster = [&](int i) {
        const uint32_t at = smem_u32(red + i);
        float v = 0.f;
        for (int c = 0; c < p.splits; ++c) {
          float u;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(mapa_shared(at, c)) : "memory");
          v += u;
        }
        return v;
      };
      for (int i = threadIdx.x; i < rows * p.M; i += Cfg::kThreads) finish(r0 + i % rows, i / rows, over_cluster);
      cluster_sync();  // every CTA's sums have been read
    }
  }
  cp_async_wait<0>();
}

// Rows n0 .. n0 + rows of W as numbers, [rows][ldd]: (code - zero) * scale, one rounding.  A
// thread per word of codes (8 numbers).
__global__ void __launch_bounds__(256) w4_expand_kernel(const W4Args p, int n0, int rows, int GPB, int odt, void* dst,
                                                        int64_t ldd) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t words = int64_t(rows) * p.blocks * 16;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < words; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / (p.blocks * 16);
    const int w = static_cast<int>(i - r * (p.blocks * 16));
    // Neighbouring threads take neighbouring k: word index j * 4 + t of the block's k order.
    const int b = w >> 4, j = (w >> 2) & 3, t = w & 3;
    const int64_t n = n0 + r;
    const int wb = w4_word_bytes(GPB, p.wide);
    const uint8_t* piece = p.data + ((n >> 4) * p.blocks + b) * w4_piece_bytes(GPB, p.wide);
    const uint32_t code = reinterpret_cast<const uint32_t*>(piece + 16 * wb + (n & 15) * 64)[t * 4 + j];
    const uint32_t* word = reinterpret_cast<const uint32_t*>(piece + (n & 15) * wb) + (j * GPB / 4) * (p.wide ? 2 : 1);
    const float s = p.wide ? __uint_as_float(word[1]) : w4_scale16(word[0], p.scale_bf16);
    const float z = float(word[0] & 15u);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = (float((code >> (4 * e)) & 15u) - z) * s;
      v[2 * e + 1] = (float((code >> (4 * e + 16)) & 15u) - z) * s;
    }
    const int64_t at = r * ldd + b * kW4Block + 32 * j + 8 * t;
    if (odt == 0) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(dst) + at);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 h;
      h.x = pack_16x2(v[0], v[1], odt == 2);
      h.y = pack_16x2(v[2], v[3], odt == 2);
      h.z = pack_16x2(v[4], v[5], odt == 2);
      h.w = pack_16x2(v[6], v[7], odt == 2);
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(dst) + at) = h;
    }
  }
}

}  // namespace tilec
