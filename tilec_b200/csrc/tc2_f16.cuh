// tc2_f16.cuh -- persistent 16-bit (bf16 / fp16) products on CTA pairs (tcgen05
// cta_group::2, kind::f16, fp32 accumulators in TMEM), sm_100a, with the epilogues of the
// language-model operators: softmax statistics, probabilities, gradients.
//
// The schedule is that of tc2_tf32p.cuh (256 x 256 tiles, two TMEM accumulators, one relay
// thread per stage in the peer CTA, bounded waits).  What differs:
//   * a stage holds 128 of K as two halves of 64 (128 bytes a row, the 128-byte swizzle's
//     width), eight MMAs of K = 16 each and one commit: at twice tf32's rate the issuing thread
//     is what runs out of time first (see the MMA role); what lies past K is neither loaded
//     nor multiplied;
//   * an operand stored along M or N (MN-major) is staged as slabs of 64 columns x 64 of K,
//     one TMA box {64, 64} each, 16-byte swizzle granules (for 16-bit types the tensor core
//     reads the plain 128-byte swizzle in either order);
//   * the number of rows (or of K, for the gradient of the weight) can come from device
//     memory: rows without a target are dropped before the product, so the host does not
//     know how many there are.  Tiles past the last row are never started;
//   * K can be cut into slices whose fp32 sums go to slabs (few tiles, long K).
//
// Where time goes (B200): 4096 x 32768 x 2048 keeps the tensor pipe 79 % (statistics) to 93 %
// busy; a tile's epilogue reads tensor memory for 1.6 us, which the next tile's MMAs cover but
// for the last tile.  Large products run into the power limit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "tc_gemm.cuh"

namespace tilec {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats rounded to nearest-even 16-bit values and packed, `lo` at the lower address.
__device__ __forceinline__ uint32_t pack_16x2(float lo, float hi, bool bf16) {
  if (bf16) return pack_bf16x2(lo, hi);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float load_16(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
              : __half2float(static_cast<const __half*>(p)[i]);
}

// What becomes of a finished tile.
enum : int {
  kEpiStats = 0,  // per row and 128-column block: (max, sum of exponentials); the target's logit
  kEpiProb = 1,   // r * (softmax - [column is the target]) in 16 bits
  kEpiAcc = 2,    // fp32 sums (a K slice's slab, or added to an earlier piece's sums)
  kEpiOut = 3,    // scale * (sums + earlier sums) in 16 bits, optionally to scattered rows
};

struct F16Args {
  int M, N, K;            // extents; one of M / K is replaced by *count when count is given
  const int* count;
  int count_is_k;
  int n_tiles, group_m, slices, kb_per_slice;
  int bf16;               // 1: bf16 operands and 16-bit outputs, 0: fp16
  const int* rows;        // row r of the product is token rows[r] (nullptr: token r)
  int col0;               // first vocabulary entry of this piece (column 0 of the product)
  // kEpiStats
  float2* part;           // [M][2 * n_tiles]: log2-domain max and sum, per 128 columns
  float* tlogit;          // [tokens]: log2(e) * logit of the target
  const int64_t* target;
  // kEpiProb
  const float2* stats;    // [tokens]: (max, sum) of the whole row
  const float* grad;      // per token (nullptr: 1)
  const float* head;      // head[1]: 1 / G with grad, see lm_ops.cuh
  float pscale;           // 1 (bf16) or 2^15 (fp16: keeps probabilities out of the subnormals)
  int m_alloc;            // rows of `out`: rows past the last one are written as zeros up to here
  // outputs
  void* out;              // 16-bit (kEpiProb, kEpiOut) or fp32 (kEpiAcc)
  int64_t ldo, slab;      // row stride (16-bit: a multiple of 8, of whole 8-column pieces) and K-slice stride
  const float* acc;       // earlier sums to add (kEpiAcc with slices == 1: may equal out), or nullptr
  int64_t ldacc;
  const float* scale;     // kEpiOut: *scale * scale2 multiplies the sums (nullptr: scale2 alone)
  float scale2;
  const void* bias;       // kEpiOut: 16-bit values added per column, or nullptr
};

struct F16Cfg {
  static constexpr int BN = 256;
  static constexpr int BK = 128;
  static constexpr int kStages = 3;
  static constexpr int kBNHalf = BN / 2;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kHalfBytes = 128 * 64 * 2;       // 64 of K of either operand's 128 rows or columns
  static constexpr int kStageBytes = 4 * kHalfBytes;     // A's two halves, then B's
  static constexpr int kStorePitch = 32;
  static constexpr int kStoreFloatsPerWarp = 32 * kStorePitch;
  static constexpr int kStoreBytes = kEpiWarps * kStoreFloatsPerWarp * 4;
  static constexpr int kBarBytes = 512;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStoreBytes + kBarBytes + 1024;
  static constexpr uint32_t kSbo = 1024u;          // 8 rows (K-major) or 8 of K (MN-major) x 128 bytes
  static constexpr uint32_t kLbo = 64 * 128u;      // MN-major: stride between 64-column slabs
  static constexpr uint32_t kTmemCols = 2 * BN;
  static_assert(kSmemBytes <= 232448, "shared memory");
  static_assert((3 * kStages + 5) * 8 + 8 <= kBarBytes, "barrier area");
};

// Bounded waits with their clock-reading loop out of line.  This kernel's roles share an SM's
// instruction caches, and the MMA thread cannot afford misses: with those loops inlined, builds
// of one source ran 12 % apart by where their code happened to lie (4096 x 32768 x 4096: 0.77
// to 0.88 ms, twice the instruction cache requests, tensor pipe 84 % busy against 67).  `hint`: how long a try may suspend the
// thread; the waits for a whole tile sleep instead of polling.
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity, uint32_t hint) {
  uint32_t ok;
  if constexpr (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(hint)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(hint)
        : "memory");
  return ok != 0;
}
__device__ __noinline__ bool mbar_poll(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t hint) {
  const unsigned long long t0 = global_ns(), limit = wait_limit();
  for (;;) {
    if (mbar_try<true>(bar, parity, hint)) return true;
    if (*abort_flag) return false;
    if (global_ns() - t0 > limit) {
      *abort_flag = 1;
      record_status(TILEC_DEV_TIMEOUT);
      return false;
    }
  }
}
constexpr uint32_t kHintStage = 64, kHintTile = 1000;  // ns
// A short loop first: entering the call costs the MMA thread more than polling (0.79 -> 0.74
// ms).  `tries`: its length, 1 where the device's limit is shortened.
__device__ __forceinline__ int wait_tries() { return wait_limit() < kWaitLimitNs ? 1 : 32; }
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_wait_far(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t hint,
                                              int tries) {
#pragma unroll 1
  for (int i = 0; i < tries; ++i)
    if (mbar_try<CLUSTER>(bar, parity, kHintStage)) return true;
  return mbar_poll(bar, parity, abort_flag, hint);
}

// Instruction descriptor for kind::f16 (format 0 = f16, 1 = bf16 for A and B alike), fp32
// accumulate; the other bits as in make_idesc_bf16.
__device__ __forceinline__ uint32_t make_idesc_16(int m, int n, bool bf16, bool a_mn, bool b_mn) {
  const uint32_t f = bf16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         ((uint32_t(n) >> 3) << 17) | ((uint32_t(m) >> 4) << 24);
}

// One warp's 32 rows x 32 columns of a tile, staged in shared memory (one row per lane's v[],
// its 16-byte pieces exchanged by the row's low bits, which keeps both passes free of bank
// conflicts), go out in 8-column pieces: four lanes cover a row's 64 (16-bit) or
// 128 (fp32) bytes.  `row_at(r)` maps staged row r to the row of `out`, or < 0 to skip it.
template <int EPI, typename RowAt>
__device__ __forceinline__ void f16_store_rows(const F16Args& p, const float* stage, RowAt row_at, int row0, int col0,
                                               float scale, int64_t slab_off, int lane) {
#pragma unroll 4
  for (int c = lane; c < 128; c += 32) {
    const int r = c >> 2, col = col0 + 8 * (c & 3);
    const int64_t orow = row_at(r);
    if (orow < 0 || col >= p.N) continue;
    const float4* staged = reinterpret_cast<const float4*>(stage + r * F16Cfg::kStorePitch);
    const float4 x0 = staged[(2 * (c & 3)) ^ (r & 7)];
    const float4 x1 = staged[(2 * (c & 3) + 1) ^ (r & 7)];
    float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    if constexpr (EPI == kEpiAcc || EPI == kEpiOut) {
      if (p.acc != nullptr) {  // rows of `acc` are padded to whole pieces
        const float4* a = reinterpret_cast<const float4*>(p.acc + static_cast<int64_t>(row0 + r) * p.ldacc + col);
        const float4 a0 = a[0], a1 = a[1];
        x[0] += a0.x; x[1] += a0.y; x[2] += a0.z; x[3] += a0.w;
        x[4] += a1.x; x[5] += a1.y; x[6] += a1.z; x[7] += a1.w;
      }
    }
    if constexpr (EPI == kEpiAcc) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.out) + slab_off + orow * p.ldo + col);
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      if constexpr (EPI == kEpiOut) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= scale;
        if (p.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < p.N) x[j] += load_16(p.bias, col + j, p.bf16);
        }
      }
      uint4 h;
      h.x = pack_16x2(x[0], x[1], p.bf16);
      h.y = pack_16x2(x[2], x[3], p.bf16);
      h.z = pack_16x2(x[4], x[5], p.bf16);
      h.w = pack_16x2(x[6], x[7], p.bf16);
      // Whole pieces: rows of `out` start and go on in steps of 16 bytes.
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.out) + orow * p.ldo + col) = h;
    }
  }
}

// Grid: 2 x P CTAs in clusters of 2 (P pairs).  A [M, K] and B [N, K], each K-major (row
// stride along M / N) or MN-major (A_MN: A stored K x M; !B_K: B stored K x N).
template <int EPI, bool A_MN, bool B_K>
__global__ void __launch_bounds__(F16Cfg::kThreads, 1)
    tc2_f16_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ F16Args p) {
  using Cfg = F16Cfg;
  constexpr int STAGES = Cfg::kStages, BK = Cfg::BK, BN = Cfg::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto a_tile = [&](int s) { return smem + s * Cfg::kStageBytes; };
  auto b_tile = [&](int s) { return smem + s * Cfg::kStageBytes + 2 * Cfg::kHalfBytes; };
  float* store_area = reinterpret_cast<float*>(smem + STAGES * Cfg::kStageBytes);
  uint8_t* bar_area = smem + STAGES * Cfg::kStageBytes + Cfg::kStoreBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(bar_area);  // [STAGES] own TMA landed
  uint64_t* empty = full + STAGES;                          // [STAGES] leader's MMAs released the stage
  uint64_t* peer_full = empty + STAGES;                     // [STAGES] (leader) the peer's TMA landed
  uint64_t* acc_full = peer_full + STAGES;                  // [2] accumulator holds a finished tile
  uint64_t* acc_empty = acc_full + 2;                       // [2] (leader) both CTAs drained it
  uint64_t* drain_bar = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (blockDim.x != Cfg::kThreads) {  // uniform across the cluster: every CTA returns
    if (threadIdx.x == 0) record_status(TILEC_DEV_BAD_LAUNCH);
    return;
  }
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&peer_full[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * Cfg::kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  __syncwarp();
  cluster_sync();  // both CTAs' barriers exist before anyone arrives remotely
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  const int tries = wait_tries();

  const int counted = p.count != nullptr ? *p.count : 0;
  const int M = p.count != nullptr && !p.count_is_k ? counted : p.M;
  const int K = p.count != nullptr && p.count_is_k ? counted : p.K;
  const int nkb_all = (K + BK - 1) / BK;
  const int mp_tiles = (M + 255) / 256;
  const int tiles = mp_tiles * p.n_tiles;
  const int total = tiles * p.slices;
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int npairs = static_cast<int>(gridDim.x >> 1);
  const int n_my = pair < total ? (total - pair + npairs - 1) / npairs : 0;

  struct TileAt {
    int m0, n0, slice, kb0, nkb;
  };
  auto tile_at = [&](int i) -> TileAt {
    int t = pair + i * npairs;
    const int slice = t / tiles;
    t -= slice * tiles;
    const int band = t / (p.group_m * p.n_tiles);
    const int first_m = band * p.group_m;
    const int band_rows = min(p.group_m, mp_tiles - first_m);
    const int in_band = t - band * p.group_m * p.n_tiles;
    const int tile_m = first_m + in_band % band_rows;
    const int tile_n = in_band / band_rows;
    const int kb0 = slice * p.kb_per_slice;
    const int nkb = max(0, min(p.kb_per_slice, nkb_all - kb0));
    return TileAt{tile_m * 256 + static_cast<int>(rank) * 128, tile_n * BN, slice, kb0, nkb};
  };

  int stored = 0;  // epilogue warps: tiles of this pair whose rows this warp has stored
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int g = 0;  // fills issued, over all tiles
      bool ok = true;
      for (int i = 0; i < n_my && ok; ++i) {
        const TileAt ta = tile_at(i);
        const int nb0 = ta.n0 + static_cast<int>(rank) * Cfg::kBNHalf;
        for (int kb = 0; kb < ta.nkb; ++kb) {
          const int s = g % STAGES;
          const uint32_t ph = (g / STAGES) & 1;
          if (!mbar_wait_far<true>(smem_u32(&empty[s]), ph ^ 1, abort_flag, kHintStage, tries)) { ok = false; break; }
          const int k0 = (ta.kb0 + kb) * BK;
          const int halves = K - k0 > 64 ? 2 : 1;
          mbar_arrive_expect_tx(&full[s], halves * 2 * Cfg::kHalfBytes);
          for (int h = 0; h < halves; ++h) {
            uint8_t* a_dst = a_tile(s) + h * Cfg::kHalfBytes;
            uint8_t* b_dst = b_tile(s) + h * Cfg::kHalfBytes;
            const int k = k0 + 64 * h;
            if constexpr (A_MN) {
#pragma unroll
              for (int j = 0; j < 2; ++j) tma_load_2d(a_dst + j * Cfg::kLbo, &tmA, &full[s], ta.m0 + 64 * j, k);
            } else {
              tma_load_2d(a_dst, &tmA, &full[s], k, ta.m0);
            }
            if constexpr (B_K) {
              tma_load_2d(b_dst, &tmB, &full[s], k, nb0);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) tma_load_2d(b_dst + j * Cfg::kLbo, &tmB, &full[s], nb0 + 64 * j, k);
            }
          }
          ++g;
        }
      }
      if (ok) {
        // Tail: the leader's release of each of the last fills has arrived before the CTA exits.
        for (int f = g - STAGES < 0 ? 0 : g - STAGES; f < g; ++f)
          if (!mbar_wait_far<true>(smem_u32(&empty[f % STAGES]), (f / STAGES) & 1, abort_flag, kHintStage, tries)) { ok = false; break; }
      }
      if (!ok) {
        for (int f = g - STAGES < 0 ? 0 : g - STAGES; f < g; ++f) mbar_drain(&full[f % STAGES], (f / STAGES) & 1);
      }
    }
  } else if (warp == 1) {
    if (leader && lane == 0) {
      // ---------------------------------------------------------- MMA issuer (leader CTA)
      // Sixteen-bit MMAs take half as long as tf32's, some 500 cycles per 64 of K, which this
      // thread's own work per stage reached first: descriptors, addresses and phases are carried
      // along instead of being built anew (4096 x 32768 x 4096: 0.905 -> 0.847 ms).
      const uint32_t idesc = make_idesc_16(256, BN, p.bf16 != 0, A_MN, !B_K);
      auto desc0 = [&](const void* tile, bool mn) {
        return make_smem_desc(smem_u32(tile), mn ? Cfg::kLbo : 16, Cfg::kSbo, kLayoutSw128);
      };
      const uint64_t a_desc = desc0(a_tile(0), A_MN), b_desc = desc0(b_tile(0), !B_K);
      constexpr uint64_t kAStep = (A_MN ? 2048 : 32) >> 4, kBStep = (B_K ? 32 : 2048) >> 4;  // K = 16
      constexpr uint64_t kHalfStep = Cfg::kHalfBytes >> 4;
      const uint32_t full_at = smem_u32(full), peer_at = smem_u32(peer_full), empty_at = smem_u32(empty);
      uint32_t s = 0, ph = 0;
      bool ok = true;
      for (int i = 0; i < n_my && ok; ++i) {
        const int b = i & 1;
        const uint32_t dcol = tmem + static_cast<uint32_t>(b * BN);
        const TileAt ta = tile_at(i);
        const int nkb = ta.nkb;
        int left = K - ta.kb0 * BK;  // of K, from this stage on
        // Buffer b last held tile i - 2: both CTAs' epilogues must have drained it.
        if (i >= 2 && !mbar_wait_far<true>(smem_u32(&acc_empty[b]), ((i >> 1) - 1) & 1, abort_flag, kHintStage, tries)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t accumulate = 0;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait_far<false>(full_at + 8 * s, ph, abort_flag, kHintStage, tries) ||
              !mbar_wait_far<true>(peer_at + 8 * s, ph, abort_flag, kHintStage, tries)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = a_desc + s * (Cfg::kStageBytes >> 4), bd = b_desc + s * (Cfg::kStageBytes >> 4);
          auto step = [&](int kk) {
            umma_bf16_pair(dcol, ad + (kk >> 2) * kHalfStep + (kk & 3) * kAStep,
                           bd + (kk >> 2) * kHalfStep + (kk & 3) * kBStep, idesc, accumulate);
            accumulate = 1;
          };
          if (left >= BK) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) step(kk);
          } else {
#pragma unroll 1
            for (int kk = 0; 16 * kk < left; ++kk) step(kk);
          }
          left -= BK;
          umma_commit_pair_both(empty_at + 8 * s);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) umma_commit_pair_both(smem_u32(&acc_full[b]));
      }
      // Every MMA issued here completes before this thread leaves its role, on every path.
      umma_commit_pair(smem_u32(drain_bar));
      mbar_drain(drain_bar, 0);
    } else if (!leader && lane == 0) {
      // ---------------------------------------------------------- relay (peer CTA)
      // The leader's MMAs read this CTA's half of each stage: tell it when the stage landed.
      const uint32_t pf = mapa_shared(smem_u32(peer_full), 0);
      int g = 0;
      bool ok = true;
      for (int i = 0; i < n_my && ok; ++i) {
        const int nkb = tile_at(i).nkb;
        for (int kb = 0; kb < nkb; ++kb, ++g) {
          const int s = g % STAGES;
          if (!mbar_wait_far<false>(smem_u32(&full[s]), (g / STAGES) & 1, abort_flag, kHintStage, tries)) { ok = false; break; }
          mbar_arrive_remote_cta(pf + static_cast<uint32_t>(s * 8));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue warps (both CTAs)
    const int e = warp - 2;
    const int q = warp & 3;  // TMEM lane quadrant of this warp: rows 32q .. 32q + 31 of the CTA's half
    const int h = e >> 2;    // which 128 of the 256 columns
    const uint32_t lane_base = static_cast<uint32_t>(32 * q) << 16;
    float* stage = store_area + e * Cfg::kStoreFloatsPerWarp;
    const uint32_t ae = mapa_shared(smem_u32(acc_empty), 0);
    float out_scale = 1.f;
    if constexpr (EPI == kEpiOut) out_scale = (p.scale != nullptr ? *p.scale : 1.f) * p.scale2;
    for (int i = 0; i < n_my; ++i) {
      const int b = i & 1;
      const TileAt ta = tile_at(i);
      const int row = ta.m0 + 32 * q + lane;  // this lane's row of the accumulator
      const int cbase = ta.n0 + h * Cfg::kBNHalf;
      // The row's constants are fetched while the MMAs still run.
      int tok = row, tcol = -1;
      float m2 = 0.f, coef = 0.f, rscale = 0.f;
      if constexpr (EPI == kEpiStats || EPI == kEpiProb) {
        if (row < M) {
          if (p.rows != nullptr) tok = p.rows[row];
          const int64_t tc = p.target[tok] - p.col0;
          tcol = tc >= cbase && tc < cbase + Cfg::kBNHalf ? static_cast<int>(tc) - cbase : -1;
          if constexpr (EPI == kEpiProb) {
            const float2 st = p.stats[tok];
            rscale = p.pscale * (p.grad != nullptr ? p.grad[tok] * p.head[1] : 1.f);
            m2 = st.x;
            coef = rscale / st.y;
          }
        }
      }
      // One answer for the warp: what follows is warp-wide.
      if (!__all_sync(0xffffffffu, mbar_wait_far<true>(smem_u32(&acc_full[b]), (i >> 1) & 1, abort_flag, kHintTile, tries)))
        break;
      tc_fence_after();
      if (i == n_my - 1) pdl_launch_dependents();
      float run_max = -INFINITY, run_sum = 0.f;
#pragma unroll 1
      for (int c = 0; c < Cfg::kBNHalf / 32; ++c) {
        const int col0 = cbase + c * 32;
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem + lane_base + static_cast<uint32_t>(b * BN + h * Cfg::kBNHalf + c * 32), r);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = ta.nkb > 0 ? __uint_as_float(r[j]) : 0.f;
        if constexpr (EPI == kEpiStats) {
          // log2 domain throughout: max and the target's logit are rounded alike, so that a
          // row whose target is its maximum has a difference of exactly zero.
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = col0 + j < p.N ? v[j] * kLog2e : -INFINITY;
          if (tcol >= c * 32 && tcol < c * 32 + 32) {
            float tl = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) tl = tcol - c * 32 == j ? v[j] : tl;
            p.tlogit[tok] = tl;
          }
          float mx = run_max;
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[j]);
          const float ref = mx == -INFINITY ? 0.f : mx;
          float sum = run_sum * ex2(run_max - ref);
#pragma unroll
          for (int j = 0; j < 32; ++j) sum += ex2(v[j] - ref);
          run_max = mx;
          run_sum = sum;
        } else {
          if constexpr (EPI == kEpiProb) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float x = ex2(fmaf(v[j], kLog2e, -m2)) * coef;
              if (tcol == c * 32 + j) x -= rscale;
              v[j] = row < M && col0 + j < p.N ? x : 0.f;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<float4*>(stage + lane * Cfg::kStorePitch)[j ^ (lane & 7)] =
                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          __syncwarp();
          const int row0 = ta.m0 + 32 * q;
          auto row_at = [&](int rr) -> int64_t {
            const int g = row0 + rr;
            if constexpr (EPI == kEpiProb) return g < p.m_alloc ? g : -1;
            if (g >= M) return -1;
            if constexpr (EPI == kEpiOut) return p.rows != nullptr ? p.rows[g] : g;
            return g;
          };
          f16_store_rows<EPI>(p, stage, row_at, row0, col0, ta.nkb > 0 ? out_scale : 0.f, ta.slice * p.slab, lane);
          __syncwarp();
        }
      }
      if constexpr (EPI == kEpiStats) {
        if (row < M) p.part[static_cast<int64_t>(row) * (2 * p.n_tiles) + (cbase >> 7)] = make_float2(run_max, run_sum);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote_cta(ae + static_cast<uint32_t>(b * 8));
      ++stored;
    }
  }

  __syncwarp();
  pdl_launch_dependents();
  tc_fence_before();
  cluster_sync();  // every remote arrive / commit targeting either CTA has landed
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, Cfg::kTmemCols);
  }
  // This CTA gave up: both CTAs' copies and MMAs have landed (cluster barrier above), so each
  // epilogue warp overwrites its block of every tile it had not stored with NaN.
  if (*abort_flag && warp >= 2) {
    const int e = warp - 2, q = warp & 3, h = e >> 2;
    const float nan = __int_as_float(0x7fc00000);
    for (int i = stored; i < n_my; ++i) {
      const TileAt ta = tile_at(i);
      const int cbase = ta.n0 + h * Cfg::kBNHalf;
      for (int rr = 0; rr < 32; ++rr) {
        const int row = ta.m0 + 32 * q + rr;
        if (row >= M) break;
        if constexpr (EPI == kEpiStats) {
          if (lane == 0)
            p.part[static_cast<int64_t>(row) * (2 * p.n_tiles) + (cbase >> 7)] = make_float2(nan, nan);
        } else {
          const int64_t orow = EPI == kEpiOut && p.rows != nullptr ? p.rows[row] : row;
          for (int c = cbase + lane; c < min(cbase + Cfg::kBNHalf, p.N); c += 32) {
            if constexpr (EPI == kEpiAcc)
              static_cast<float*>(p.out)[ta.slice * p.slab + orow * p.ldo + c] = nan;
            else
              static_cast<unsigned short*>(p.out)[orow * p.ldo + c] = 0x7fff;
          }
        }
      }
    }
  }
}

}  // namespace tilec
