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
// The codes are streamed once (K/2 bytes a row of W) for up to 16 rows of 16-bit x and 8 of fp32 x,
// and once per 128 rows for up to 256 rows of 16-bit x whose type the scales share; for the rest W
// is expanded in memory first (w4_expand_kernel, 5 times the codes' bytes in 16 bits, 9 in fp32,
// written and read again).  At full
// bandwidth an SM has under three lane-instructions per weight, too few to convert and multiply
// each weight on the FMA pipe, so the sums run on tensor cores: mma.sync, 16 rows of W against 8
// columns at a time, for up to 16 rows of x (w4_stream.cuh), tcgen05 with the weight expanded in
// shared memory for more (w4_tc.cuh).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tilec {

constexpr int kW4Block = 128;  // k per 64-byte block of codes

struct W4Args {
  const uint8_t* data;     // [row tiles][blocks][piece]
  int wide;                // fp32 scales: (zero, scale) pairs
  int scale_bf16;          // 16-bit scales: bf16 (else fp16)
  int N, K, blocks;
  const void* x;           // [M][ldx] of type dtype
  int64_t ldx;
  int dtype;               // TILEC_DTYPE_* of x, bias and out
  int M, cols;             // cols: M, or M times the digits or terms of w4_stream_kernel
  int vec_x;               // 16-byte loads of x allowed (16-bit types)
  void* out;               // [M][ldo]
  int64_t ldo;
  const void* bias;        // [N] or nullptr
  int splits;              // CTAs of a cluster that share a row tile's K
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

// The pair of codes i of a word, minus the zero point (zm = the magic number | zero, twice): the
// well-known way to a 16-bit float, a small number in the low bits of the mantissa of a power of two.
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
