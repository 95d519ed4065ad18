// w4_tc.cuh -- products of some tens of rows with 4-bit weights on the 5th-generation tensor
// cores (tcgen05, fp32 accumulators in TMEM), the weight expanded on the way.
//
// From some 9 to 17 rows of x on (see plan_w4), mma.sync's share of the work grows with the rows
// while the weight still has to be read once (129 to 256 rows: twice, 128 rows at a time); expanding it in HBM first (w4_expand_kernel) costs five times its bytes.
// Here a CTA takes 128 rows of W as the M side of the product and up to 128 rows of x as its N
// side (swapped, so that the few rows of x pad to 16 and not to 128 or 256):
//   * one warp fetches codes (bulk copies of four blocks per 16-row tile, a run of memory each,
//     a lane each: an SM starts one some 55 ns after another, so two blocks a copy were too
//     few) and x (TMA boxes of 64 k x rows, 128-byte swizzle) into rings;
//   * 16 warps expand: 8 codes of a row become one 16-byte piece of the K-major operand tile,
//     (code - zero) exactly, times the scale with one rounding to x's type, and go where the
//     swizzle wants them.  Two groups of 8 warps take alternate blocks, into two buffers;
//   * one thread issues the MMAs (M = 128, N = rows of x, K = 16);
//   * the same 16 warps read the accumulator and store: lanes are rows of W, so a warp stores
//     32 neighbouring outputs of one row of x.
// K is split over CTAs that write fp32 slabs (f16_join_slabs_kernel adds them in order).
//
// Measured (graph replay): 4096 x 4096 12 us for 32 rows, 15 for 128; 8192 x 8192 26.5 and 39
// (the codes alone: 6 at HBM's rate); 28672 x 8192 84 and 128.  A CTA takes some 0.65 us per
// block: the busier SMs issue 54 % of the time, three or four operand buffers and three code
// stages are no faster, and a last wave of tiles that fills half the SMs is the rest.
#pragma once

#include "w4_stream.cuh"

namespace tilec {

struct W4TcArgs {
  W4Args w;
  int n_cols;          // rows of x rounded up to 16
  int per_cta;         // blocks of K a CTA takes (even)
  float* slabs;        // splits > 1: [split][M][lds]
  int64_t lds;
};

template <int GPB>
struct W4TcCfg {
  static constexpr int kExpandWarps = 16;
  static constexpr int kThreads = 64 + 32 * kExpandWarps;
  static constexpr int kRows = 128;
  static constexpr int kMaxCols = 128;
  static constexpr int kPiece = w4_piece_bytes(GPB, false);
  static constexpr int kRun = 4;                               // blocks a copy
  static constexpr int kCodeTile = kRun * kPiece;              // of one 16-row tile
  static constexpr int kCodeStage = 8 * kCodeTile;
  static constexpr int kCodeStages = 2;
  static constexpr int kHalf = kRows * 128;                    // 64 of K, K-major
  static constexpr int kABytes = 2 * kHalf;                    // a block
  static constexpr int kMaxBStages = 8;
  static constexpr int kBBytes = 65536;                        // x: as many blocks as fit, up to 8
  static constexpr int kABufs = 2;   // three or four: no faster (28672 x 8192, 32 rows: 84, 86, 88 us)
  static constexpr int kOffB = kABufs * kABytes, kOffCodes = kOffB + kBBytes;
  static constexpr int kOffBars = kOffCodes + kCodeStages * kCodeStage;
  static constexpr int kBarBytes = 256;
  static constexpr int kSmemBytes = kOffBars + kBarBytes + 1024;
  static_assert(kSmemBytes <= 232448 && kOffBars % 16 == 0, "shared memory");
};

// D[tmem] (+)= A[smem desc] * B[smem desc], kind::f16, one CTA.
__device__ __forceinline__ void umma_16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t mul_16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF16)
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Grid: x = 128-row tiles * splits.  The scales are of x's type (a product of two such numbers
// rounds once).
template <bool BF16, int GPB>
__global__ void __launch_bounds__(W4TcCfg<GPB>::kThreads, 1)
    w4_tc_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ W4TcArgs a) {
  using Cfg = W4TcCfg<GPB>;
  constexpr int WB = w4_word_bytes(GPB, false), SC = Cfg::kCodeStages, RUN = Cfg::kRun, NA = Cfg::kABufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a_buf = smem;                        // [NA][kABytes]
  uint8_t* b_buf = smem + Cfg::kOffB;           // [SB][half][n_cols][128]
  uint8_t* codes = smem + Cfg::kOffCodes;       // [SC][16-row tile][kCodeTile]
  uint64_t* c_full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBars);
  uint64_t* c_empty = c_full + SC;
  uint64_t* b_full = c_empty + SC;
  uint64_t* b_empty = b_full + Cfg::kMaxBStages;
  uint64_t* a_full = b_empty + Cfg::kMaxBStages;   // [NA]
  uint64_t* a_empty = a_full + NA;   // [NA]
  uint64_t* acc_full = a_empty + NA;
  uint64_t* drain_bar = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const W4Args& p = a.w;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockDim.x != Cfg::kThreads) {
    if (threadIdx.x == 0) record_status(TILEC_DEV_BAD_LAUNCH);
    return;
  }
  const int tile = static_cast<int>(blockIdx.x) / p.splits, split = static_cast<int>(blockIdx.x) - tile * p.splits;
  const int n0 = tile * Cfg::kRows;
  const int b_begin = min(p.blocks, split * a.per_cta), b_end = min(p.blocks, b_begin + a.per_cta);
  const int nblk = b_end - b_begin;
  const uint32_t b_half = static_cast<uint32_t>(a.n_cols) * 128;  // bytes of x per 64 k
  const int SB = min(Cfg::kMaxBStages, static_cast<int>(Cfg::kBBytes / (2 * b_half)));
  const uint32_t tmem_cols = a.n_cols <= 32 ? 32 : a.n_cols <= 64 ? 64 : 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SC; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], Cfg::kExpandWarps / 2 * RUN);
    }
    for (int s = 0; s < Cfg::kMaxBStages; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int s = 0; s < NA; ++s) {
      mbar_init(&a_full[s], Cfg::kExpandWarps / 2);
      mbar_init(&a_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  const int tries = wait_tries();

  bool ok = true;
  if (warp == 0) {
    // ------------------------------------------------------------ fetching warp
    const int row_tiles = min(8, (p.N - n0 + 15) / 16);
    const uint8_t* src =
        p.data + ((static_cast<int64_t>(tile) * 8 + min(lane, row_tiles - 1)) * p.blocks + b_begin) * Cfg::kPiece;
    int i = 0, units = 0, bs = 0;  // blocks of x and units of codes that were sent for
    uint32_t b_phase = 1;
    for (; i < nblk && ok; ++i) {
      if (i % RUN == 0) {  // codes of this block and the next ones
        const int u = i / RUN, s = u % SC, run = min(RUN, nblk - i);
        ok = __all_sync(0xffffffffu, u < SC || mbar_wait(&c_empty[s], ((u / SC) - 1) & 1, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&c_full[s], static_cast<uint32_t>(row_tiles * run * Cfg::kPiece));
        __syncwarp();
        if (lane < row_tiles)
          bulk_load(codes + s * Cfg::kCodeStage + lane * Cfg::kCodeTile, src + static_cast<int64_t>(i) * Cfg::kPiece,
                    run * Cfg::kPiece, &c_full[s]);
        units = u + 1;
      }
      ok = __all_sync(0xffffffffu, i < SB || mbar_wait(&b_empty[bs], b_phase, abort_flag));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&b_full[bs], 2 * b_half);
        for (int h = 0; h < 2; ++h)
          tma_load_2d(b_buf + (2 * bs + h) * b_half, &tm_x, &b_full[bs], (b_begin + i) * kW4Block + 64 * h, 0);
      }
      if (++bs == SB) {
        bs = 0;
        b_phase ^= 1;
      }
    }
    // Every copy has landed before this CTA may end, on every path (a unit's codes go out before
    // the wait for its first block's room in the ring of x, which may be given up).
    if (lane == 0) {
      for (int f = max(0, units - SC); f < units; ++f) mbar_drain(&c_full[f % SC], (f / SC) & 1);
      for (int f = max(0, i - SB); f < i; ++f) mbar_drain(&b_full[f % SB], (f / SB) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = make_idesc_16(128, a.n_cols, BF16, false, false);
      // Descriptors and addresses are carried along: this thread's own work per block counts.
      const uint64_t a_desc = make_smem_desc(smem_u32(a_buf), 16, 1024, kLayoutSw128);
      const uint64_t b_desc = make_smem_desc(smem_u32(b_buf), 16, 1024, kLayoutSw128);
      const uint32_t af = smem_u32(a_full), bf = smem_u32(b_full);
      uint32_t s = 0, b_phase = 0, buf = 0, a_phase = 0, accumulate = 0;
      for (int i = 0; i < nblk; ++i) {
        if (!mbar_wait_far<false>(bf + 8 * s, b_phase, abort_flag, kHintStage, tries) ||
            !mbar_wait_far<false>(af + 8 * buf, a_phase, abort_flag, kHintStage, tries)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = a_desc + buf * (Cfg::kABytes >> 4), bd = b_desc + s * (b_half >> 3);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          umma_16(tmem, ad + (kk >> 2) * (Cfg::kHalf >> 4) + (kk & 3) * 2, bd + (kk >> 2) * (b_half >> 4) + (kk & 3) * 2, idesc,
                  accumulate);
          accumulate = 1;
        }
        umma_commit(&a_empty[buf]);
        umma_commit(&b_empty[s]);
        if (++buf == NA) {
          buf = 0;
          a_phase ^= 1;
        }
        if (++s == static_cast<uint32_t>(SB)) {
          s = 0;
          b_phase ^= 1;
        }
      }
      if (ok) umma_commit(acc_full);
      umma_commit(drain_bar);  // every MMA issued here completes before this thread goes on
      mbar_drain(drain_bar, 0);
    }
  } else {
    // ------------------------------------------------------------ expanding, then storing warps
    const int e = warp - 2, group = e >> 3;  // blocks group, group + 2, ...
    const int g = lane >> 2, t = lane & 3;
    // Rows of the 16-row tile: pairs of lane groups whose codes and operand pieces lie in
    // different banks.
    const int row = (g & 1) ? (g >> 1) ^ 5 : g >> 1;
    const uint32_t rt = e & 7;
    uint32_t magic;
    asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300u : 0x64006400u));
    for (int i = group; i < nblk; i += 2) {
      const int u = i / RUN, s = u % SC, buf = i % NA;
      ok = __all_sync(0xffffffffu, mbar_wait(&c_full[s], (u / SC) & 1, abort_flag) &&
                                       (i < NA || mbar_wait(&a_empty[buf], ((i / NA) - 1) & 1, abort_flag)));
      if (!ok) break;
      const uint32_t piece = smem_u32(codes) + s * Cfg::kCodeStage + rt * Cfg::kCodeTile + (i % RUN) * Cfg::kPiece;
      const uint32_t dst = smem_u32(a_buf) + buf * Cfg::kABytes + (16 * rt + row) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // row, row + 8
        const uint4 q = lds128(piece + 16 * WB + (row + 8 * h) * 64 + t * 16);
        uint32_t words[WB / 4];
        lds_words(words, piece + (row + 8 * h) * WB);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t word = words[j * GPB / 4];
          const uint32_t zm = magic | __byte_perm(word, 0, 0x1010), sc = __byte_perm(word, 0, 0x3232);
          const uint32_t w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
          uint32_t v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = mul_16x2<BF16>(w4_pair<BF16>(w, k, magic, zm), sc);
          // Piece 4j + t of the row's 16: half j >> 1, exchanged by the row's low bits.
          const uint32_t chunk = (4 * (j & 1) + t) ^ (row & 7);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + h * 1024 + (j >> 1) * Cfg::kHalf +
                                                                         chunk * 16),
                       "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                       : "memory");
        }
      }
      fence_proxy_async_smem();  // the MMAs read what was just stored
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&a_full[buf]);
        mbar_arrive(&c_empty[s]);
      }
    }
    if (ok) ok = __all_sync(0xffffffffu, nblk == 0 || mbar_wait(acc_full, 0, abort_flag));
    tc_fence_after();
    const int q = warp & 3, col0 = (e >> 2) * 32;  // TMEM lanes 32q .., 32 columns
    const int n = n0 + 32 * q + lane;
    if (col0 < a.n_cols) {
      uint32_t r[32];
      if (nblk > 0 && ok) {
        tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(32 * q) << 16) + col0, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = ok ? 0u : 0x7fc00000u;  // gave up: NaN
      }
      if (n < p.N) {
        const float bias = p.splits == 1 && p.bias != nullptr ? load_16(p.bias, n, BF16) : 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int m = col0 + j;
          if (m >= p.M) break;
          const float v = __uint_as_float(r[j]);
          if (p.splits > 1)
            a.slabs[(static_cast<int64_t>(split) * p.M + m) * a.lds + n] = v;
          else
            store_from_float(p.out, int64_t(m) * p.ldo + n, BF16 ? 2 : 1, v + bias);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

}  // namespace tilec
