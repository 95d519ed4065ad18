// w4.cuh -- products with 4-bit weights: y[m, n] = sum_k x[m, k] * (code[n, k] - zero) * scale,
// scale and zero per group of consecutive k.
//
// Layout of the codes (made once by the caller): rows of 64-byte blocks, a block holding 128
// consecutive k.  Word 4t + j of a block (t, j = 0..3) holds k = 32j + 8t + 0..7, the even
// ones of these in nibbles 0..3 and the odd ones in nibbles 4..7.  So
//   * lane t of the four lanes that share a row loads its words t*4 .. t*4+3 as 16 bytes;
//   * word j of all four lanes covers k = 32j .. 32j+31, i.e. one group even when groups are
//     32 long, and feeds two tensor-core steps of K = 16;
//   * (word >> 4i) & 0x000F000F is the pair k = 2i, 2i+1, next to each other as x is.
// Scales (and zero points) lie [group][n]: a warp's rows are neighbours.
//
// Few rows of x: the product streams the codes once (K/2 bytes a row of W) and is bound by
// memory.  Per byte of codes an SM has about 2.8 x 32 lane-instructions per weight pair at
// full bandwidth, too few to convert and multiply each weight on the FMA pipe, so the sums
// run on mma.sync m16n8k16: 16 rows of W against up to 8 columns (tokens) at a time, fp32
// accumulators.  (tcgen05 would need the converted weights to pass through shared memory
// first; with 8 columns its rate is not what bounds this.)  A code becomes a 16-bit float
// exactly: 0x4300 | code is 128 + code in bf16 (0x6400 | code is 1024 + code in fp16), minus
// (128 + zero).  Products are exact, sums fp32; the scale multiplies a group's fp32 sum.
// fp32 x is cut into three bf16 parts (8 bits each, exact), three columns per token.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tilec {

constexpr int kW4Warps = 8;
constexpr int kW4Block = 128;  // k per 64-byte block of codes

struct W4Args {
  const uint4* codes;   // [N][blocks * 4]
  const void* scales;   // [groups][N], type sdt
  const uint8_t* zeros; // [groups][N] or nullptr (zero = 8)
  int sdt;              // TILEC_DTYPE_*
  int N, blocks;
  int group_blocks;     // blocks per group (groups of 128 and more)
  const unsigned short* x;  // [cols][ldx], 16-bit, readable up to blocks * 128
  int64_t ldx;
  int cols;             // columns: rows of x times parts
  int parts;            // 1, or 3 for fp32 x
  int M;
  void* out;            // [M][ldo] of type odt
  int64_t ldo;
  int odt;
  const void* bias;     // [N] of type odt, or nullptr
  int splits;           // CTAs of a cluster that share a row tile's K
};

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dt) {
  if (dt == 0) return static_cast<const float*>(p)[i];
  if (dt == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int64_t i, int dt, float v) {
  if (dt == 0)
    static_cast<float*>(p)[i] = v;
  else if (dt == 1)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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
template <bool BF16>
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, int i, uint32_t zm) {
  constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
  const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | kMagic;
  uint32_t r;
  if constexpr (BF16)
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zm));
  else
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(zm));
  return r;
}

// A block computes 16 * MT rows of W for 8 * NT columns; its warps (and the cluster's CTAs)
// take 128-k blocks in turn, so that neighbours read neighbouring 64 bytes of a row, and add
// their sums in a fixed order.  GPB: scale groups per 128-k block (4, 2, or 1 for longer
// groups).  Grid: x = row tiles * splits, clusters of `splits` along x.
template <bool BF16, int NT, int MT, int GPB>
__global__ void __launch_bounds__(32 * kW4Warps) w4_mma_kernel(const __grid_constant__ W4Args p) {
  constexpr int U = MT == 1 ? 4 : 2;  // blocks in flight per warp
  constexpr int ROWS = 16 * MT, COLS = 8 * NT;
  __shared__ float red[kW4Warps][ROWS][COLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / p.splits * ROWS;
  const int step = kW4Warps * p.splits;
  pdl_wait();
  pdl_launch_dependents();

  const uint4* row_ptr[2 * MT];
  int row[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    row[i] = min(n0 + g + 8 * i, p.N - 1);
    row_ptr[i] = p.codes + static_cast<int64_t>(row[i]) * p.blocks * 4 + t;
  }
  const unsigned short* xp[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int col = 8 * i + g;
    xp[i] = col < p.cols ? p.x + static_cast<int64_t>(col) * p.ldx + 8 * t : nullptr;
  }
  float total[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) total[m][i][j] = 0.f;

  constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
  for (int b0 = rank * kW4Warps + warp; b0 < p.blocks; b0 += U * step) {
    uint4 q[U][2 * MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * step;
      if (b < p.blocks) {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) q[u][i] = __ldcs(row_ptr[i] + static_cast<int64_t>(b) * 4);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * step;
      if (b >= p.blocks) break;
      float acc[MT][NT][4];
      uint32_t zm[2 * MT];
      float sc[2 * MT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j % (4 / GPB) == 0) {
          const int64_t grp = GPB > 1 ? int64_t(b) * GPB + j / (4 / GPB)
                                      : (p.group_blocks == 1 ? b : b / p.group_blocks);
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) {
            sc[i] = load_as_float(p.scales, grp * p.N + row[i], p.sdt);
            zm[i] = kMagic | (p.zeros != nullptr ? uint32_t(p.zeros[grp * p.N + row[i]]) * 0x10001u : 0x00080008u);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m][i][e] = 0.f;
        }
        uint4 xv[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i)
          xv[i] = xp[i] != nullptr ? *reinterpret_cast<const uint4*>(xp[i] + static_cast<int64_t>(b) * kW4Block + 32 * j)
                                   : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 qa = q[u][2 * m], qb = q[u][2 * m + 1];
          const uint32_t wa = j == 0 ? qa.x : j == 1 ? qa.y : j == 2 ? qa.z : qa.w;
          const uint32_t wb = j == 0 ? qb.x : j == 1 ? qb.y : j == 2 ? qb.z : qb.w;
          uint32_t a[4], c[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i] = w4_pair<BF16>(wa, i, zm[2 * m]);
            c[i] = w4_pair<BF16>(wb, i, zm[2 * m + 1]);
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            mma_16816<BF16>(acc[m][i], a[0], c[0], a[1], c[1], xv[i].x, xv[i].y);
            mma_16816<BF16>(acc[m][i], a[2], c[2], a[3], c[3], xv[i].z, xv[i].w);
          }
        }
        if ((j + 1) % (4 / GPB) == 0) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
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
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(&red[warp][16 * m + g][8 * i + 2 * t]) = make_float2(total[m][i][0], total[m][i][1]);
      *reinterpret_cast<float2*>(&red[warp][16 * m + g + 8][8 * i + 2 * t]) = make_float2(total[m][i][2], total[m][i][3]);
    }
  __syncthreads();
  float* sums = &red[0][0][0];
  for (int i = threadIdx.x; i < ROWS * COLS; i += 32 * kW4Warps) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kW4Warps; ++w) s += (&red[w][0][0])[i];
    sums[i] = s;  // element i of red[0] is read by this thread alone
  }
  if (p.splits > 1) {
    cluster_sync();
    if (rank == 0) {
      for (int i = threadIdx.x; i < ROWS * COLS; i += 32 * kW4Warps) {
        float s = sums[i];
        for (int r = 1; r < p.splits; ++r) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(sums + i), r)) : "memory");
          s += v;
        }
        sums[i] = s;
      }
    }
    cluster_sync();  // the other CTAs' sums have been read
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  for (int i = threadIdx.x; i < ROWS * p.M; i += 32 * kW4Warps) {
    const int r = i % ROWS, m = i / ROWS, n = n0 + r;
    if (n >= p.N) continue;
    float v = 0.f;
    for (int k = p.parts - 1; k >= 0; --k) v += sums[r * COLS + m * p.parts + k];  // smallest part first
    if (p.bias != nullptr) v += load_as_float(p.bias, n, p.odt);
    store_from_float(p.out, int64_t(m) * p.ldo + n, p.odt, v);
  }
}

// Columns for w4_mma_kernel: x rows padded with zeros to whole 128-k blocks; an fp32 row
// becomes three bf16 rows whose sum it is (each takes the upper half of what is left, so
// nothing overflows; what is not finite stays whole in the first).  A block per row and
// 256 * 8 elements.
__global__ void __launch_bounds__(256) w4_columns_kernel(const void* __restrict__ x, int64_t ldx, int K, int f32,
                                                         unsigned short* __restrict__ dst, int64_t ldd) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t m = blockIdx.y;
  const int k0 = (static_cast<int>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (k0 >= ldd) return;
  if (!f32) {
    const unsigned short* s = static_cast<const unsigned short*>(x) + m * ldx;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < K) w[j >> 1] |= uint32_t(s[k0 + j]) << (16 * (j & 1));
    *reinterpret_cast<uint4*>(dst + m * ldd + k0) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  const float* s = static_cast<const float*>(x) + m * ldx;
  uint32_t w[3][4] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float v = k0 + j < K ? s[k0 + j] : 0.f;
    const bool finite = fabsf(v) < INFINITY;
    if (v != v) v = __int_as_float(0x7fc00000);
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      const uint32_t top = __float_as_uint(v) & 0xFFFF0000u;
      w[part][j >> 1] |= (top >> 16) << (16 * (j & 1));
      v = finite ? v - __uint_as_float(top) : 0.f;
    }
  }
#pragma unroll
  for (int part = 0; part < 3; ++part)
    *reinterpret_cast<uint4*>(dst + (m * 3 + part) * ldd + k0) =
        make_uint4(w[part][0], w[part][1], w[part][2], w[part][3]);
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
    const uint32_t code = reinterpret_cast<const uint32_t*>(p.codes + (n0 + r) * p.blocks * 4)[b * 16 + t * 4 + j];
    const int64_t grp = GPB > 1 ? int64_t(b) * GPB + j * GPB / 4 : b / p.group_blocks;
    const float s = load_as_float(p.scales, grp * p.N + n0 + r, p.sdt);
    const float z = p.zeros != nullptr ? float(p.zeros[grp * p.N + n0 + r]) : 8.f;
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
