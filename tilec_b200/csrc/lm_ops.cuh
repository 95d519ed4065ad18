// lm_ops.cuh -- host side and C ABI of the language-model operators (part of the library's
// single translation unit, after tilec_mm.cu's own host code).
#pragma once

namespace tilec {
namespace {

constexpr int64_t kW4MaxSmem = 232448;    // shared memory a CTA may have

// ---------------------------------------------------------------- 16-bit products
struct LmInfo {
  int f16_slots = 0;  // CTA pairs of tc2_f16_kernel resident at once
  cudaError_t err = cudaSuccess;
};
LmInfo g_lm[kMaxDevices];
std::once_flag g_lm_once[kMaxDevices];

int lm_device(DeviceInfo** d, LmInfo** lm) {
  const int rc = current_device(d);
  if (rc) return rc;
  const int dev = (*d)->dev;
  std::call_once(g_lm_once[dev], [dev]() {
    LmInfo& m = g_lm[dev];
    auto acc = [&](cudaError_t e) {
      if (m.err == cudaSuccess) m.err = e;
    };
    auto attr = [&](auto kern) {
      acc(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F16Cfg::kSmemBytes));
    };
    attr(tc2_f16_kernel<kEpiStats, false, true>);
    attr(tc2_f16_kernel<kEpiProb, false, true>);
    attr(tc2_f16_kernel<kEpiOut, false, false>);
    attr(tc2_f16_kernel<kEpiAcc, false, false>);
    attr(tc2_f16_kernel<kEpiOut, true, false>);
    attr(tc2_f16_kernel<kEpiAcc, true, false>);
    attr(tc2_f16_kernel<kEpiOut, false, true>);
    attr(tc2_f16_kernel<kEpiAcc, false, true>);
    auto w4_attr = [&](auto kern) {
      acc(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kW4MaxSmem)));
    };
    auto w4_attrs = [&](auto gpb, auto wide) {
      constexpr int G = decltype(gpb)::value;
      constexpr bool W = decltype(wide)::value;
      if constexpr (W) {
        w4_attr(w4_stream_kernel<1, G, TILEC_DTYPE_F32, 0>);
      } else {
        w4_attr(w4_stream_kernel<1, G, TILEC_DTYPE_F16, 0>);
        w4_attr(w4_stream_kernel<1, G, TILEC_DTYPE_BF16, 0>);
      }
      w4_attr(w4_stream_kernel<1, G, W ? 0 : 1, kW4Terms>);
      w4_attr(w4_stream_kernel<3, G, W ? 0 : 1, kW4Terms>);
      w4_attr(w4_stream_kernel<1, G, W ? 0 : 1, TILEC_DTYPE_F16>);
      w4_attr(w4_stream_kernel<1, G, W ? 0 : 1, TILEC_DTYPE_BF16>);
      w4_attr(w4_stream_kernel<2, G, W ? 0 : 1, TILEC_DTYPE_F16>);
      w4_attr(w4_stream_kernel<2, G, W ? 0 : 1, TILEC_DTYPE_BF16>);
    };
    auto w4_all = [&](auto gpb) {
      constexpr int G = decltype(gpb)::value;
      w4_attr(w4_tc_kernel<true, G>);
      w4_attr(w4_tc_kernel<false, G>);
      w4_attrs(gpb, std::true_type{});
      w4_attrs(gpb, std::false_type{});
    };
    w4_all(std::integral_constant<int, 1>{});
    w4_all(std::integral_constant<int, 2>{});
    w4_all(std::integral_constant<int, 4>{});
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(2, 1, 1);
    lc.blockDim = dim3(F16Cfg::kThreads);
    lc.dynamicSmemBytes = F16Cfg::kSmemBytes;
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = 2;
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
    lc.attrs = &a;
    lc.numAttrs = 1;
    acc(cudaOccupancyMaxActiveClusters(&m.f16_slots, tc2_f16_kernel<kEpiOut, false, false>, &lc));
    if (m.err == cudaSuccess && m.f16_slots < 1) m.err = cudaErrorLaunchOutOfResources;
    cudaGetLastError();
  });
  if (g_lm[dev].err != cudaSuccess) return TILEC_ERR_NO_DEVICE;
  *lm = &g_lm[dev];
  return TILEC_OK;
}

// A 16-bit matrix of `outer` rows of `inner` elements, row stride ld (a multiple of 8, base
// 16-byte aligned), read in boxes of 64 x box_out; out-of-range elements read as zero.
int encode16(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int64_t ld, int box_out, bool bf16) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = get_encode();
  if (!enc) return TILEC_ERR_NO_DEVICE;
  cuuint64_t dims[2] = {cuuint64_t(inner), cuuint64_t(outer)};
  cuuint64_t strides[1] = {cuuint64_t(ld) * 2};
  cuuint32_t box[2] = {64, cuuint32_t(box_out)};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TILEC_OK
             : TILEC_ERR_BAD_ARG;
}

// One operand: M (or N) x K, stored row-major (mn = false) or as its transpose (mn = true).
struct Op16 {
  const void* p;
  int64_t ld;
  bool mn;
};

template <int EPI, bool A_MN, bool B_K>
int launch_f16(const Op16& A, const Op16& B, int64_t M, int64_t N, int64_t K, F16Args p, const LmInfo& lm,
               cudaStream_t s) {
  CUtensorMap ma, mb;
  const bool bf16 = p.bf16 != 0;
  int rc = A_MN ? encode16(&ma, A.p, M, K, A.ld, 64, bf16) : encode16(&ma, A.p, K, M, A.ld, 128, bf16);
  if (rc) return rc;
  rc = B_K ? encode16(&mb, B.p, K, N, B.ld, 128, bf16) : encode16(&mb, B.p, N, K, B.ld, 64, bf16);
  if (rc) return rc;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.n_tiles = static_cast<int>(cdiv(N, 256));
  p.group_m = 16;
  if (p.slices <= 1) {
    p.slices = 1;
    p.kb_per_slice = static_cast<int>(cdiv(K, F16Cfg::BK));
  }
  const int64_t total = cdiv(M, 256) * p.n_tiles * p.slices;
  if (total >= (int64_t(1) << 30)) return TILEC_ERR_UNSUPPORTED;
  const int pairs = static_cast<int>(total < lm.f16_slots ? total : lm.f16_slots);
  return launch_k(tc2_f16_kernel<EPI, A_MN, B_K>, dim3(static_cast<unsigned>(2 * pairs)), dim3(F16Cfg::kThreads),
                  F16Cfg::kSmemBytes, s, 2, ma, mb, p);
}

// K slices of a product of few tiles: as many as fill the CTA pairs once, each at least
// four stages (512) deep.
int f16_slices(int64_t M, int64_t N, int64_t K, const LmInfo& lm, int* kb_per_slice) {
  const int64_t tiles = cdiv(M, 256) * cdiv(N, 256), nkb = cdiv(K, F16Cfg::BK);
  int64_t n = lm.f16_slots / tiles;
  if (n > nkb / 4) n = nkb / 4;
  if (n < 1) n = 1;
  const int64_t per = cdiv(nkb, n);
  *kb_per_slice = static_cast<int>(per);
  return static_cast<int>(cdiv(nkb, per));
}

#define TILEC_TRY(expr)            \
  do {                             \
    const int rc_ = (expr);        \
    if (rc_) return rc_;           \
  } while (0)

// A 16-bit product with its sums in fp32: K slices go through slabs ([slices][M][lda] floats),
// a sum over several products (dx over pieces of the vocabulary) through acc_in / acc_out
// ([M][lda] floats).  out == nullptr: the sums stay in acc_out.  `odd`: room for M rows of lda
// 16-bit values, where out's rows are not made of whole 16-byte pieces and slices == 1.
inline bool odd_rows(const void* out, int64_t ldo, int64_t N) {
  return !aligned16(out) || ldo % 8 != 0 || N % 8 != 0;
}

template <bool A_MN, bool B_K>
int product16(const Op16& A, const Op16& B, int64_t M, int64_t N, int64_t K, F16Args a, int slices, int kb,
              int64_t lda, const float* acc_in, float* acc_out, void* out, int64_t ldo, float* slabs,
              void* odd, const LmInfo& lm, const DeviceInfo& d, cudaStream_t s) {
  a.slices = slices;
  a.kb_per_slice = kb;
  if (slices > 1) {
    F16Args b = a;
    b.out = slabs;
    b.ldo = lda;
    b.slab = M * lda;
    b.acc = nullptr;
    TILEC_TRY((launch_f16<kEpiAcc, A_MN, B_K>(A, B, M, N, K, b, lm, s)));
    int64_t blocks = cdiv(M * cdiv(N, 8), 256);
    if (blocks > int64_t(d.sms) * 8) blocks = int64_t(d.sms) * 8;
    return launch_k(f16_join_slabs_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1,
                    static_cast<const float*>(slabs), slices, b.slab, lda, acc_in, acc_out,
                    static_cast<unsigned short*>(out), ldo, M, N, a.count_is_k ? nullptr : a.count, a.rows, a.scale,
                    a.scale2, a.bias, a.bf16, odd_rows(out, ldo, N) ? 0 : 1);
  }
  a.acc = acc_in;
  a.ldacc = lda;
  if (out == nullptr) {
    a.out = acc_out;
    a.ldo = lda;
    return launch_f16<kEpiAcc, A_MN, B_K>(A, B, M, N, K, a, lm, s);
  }
  if (!odd_rows(out, ldo, N)) {
    a.out = out;
    a.ldo = ldo;
    return launch_f16<kEpiOut, A_MN, B_K>(A, B, M, N, K, a, lm, s);
  }
  const int* rows = a.rows;
  const int* count = a.count_is_k ? nullptr : a.count;
  a.rows = nullptr;
  a.out = odd;
  a.ldo = lda;
  TILEC_TRY((launch_f16<kEpiOut, A_MN, B_K>(A, B, M, N, K, a, lm, s)));
  const int dense = rows == nullptr && ldo == N && aligned16(out);
  int64_t blocks = cdiv(M * N, dense ? 2048 : 256);
  if (blocks > int64_t(d.sms) * 16) blocks = int64_t(d.sms) * 16;
  return launch_k(unpad16_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1,
                  static_cast<const unsigned short*>(odd), lda, static_cast<unsigned short*>(out), ldo, M,
                  static_cast<int>(N), count, rows, dense);
}

// ---------------------------------------------------------------- linear cross entropy
// Bytes of probabilities (16-bit) or logits (fp32) of one piece of the vocabulary.
constexpr int64_t kCePieceBytes = int64_t(512) << 20;
constexpr int64_t kCePieceMin = 4096;

struct CeCall {
  const void* x;
  const void* w;
  const int64_t* target;
  int dtype;
  int64_t T, V, D, ldx, ldw, ignore;
  int reduction;
};

struct CePlan {
  bool f32 = false, bf16 = false;
  bool compact = false, pack_x = false, pack_w = false;
  int64_t dp = 0;                // row stride of packed 16-bit operands
  int64_t piece = 0, pieces = 0; // vocabulary entries per piece
  int64_t ldp = 0;               // row stride of a piece's probabilities / logits
  int64_t nblk = 0;              // partial statistics per row
  int64_t ldacc = 0;             // row stride of fp32 sums of dx
  int dx_slices = 1, dx_kb = 0, dw_slices = 1, dw_kb = 0;
  size_t off_head = 0, off_rows = 0, off_x = 0, off_w = 0, off_part = 0, off_tlogit = 0, off_loss = 0, off_p = 0,
         off_acc = 0, off_slabs = 0, off_odd = 0, off_mm = 0;
  size_t mm_bytes = 0, bytes = 0;
};

inline bool rows_aligned16(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

Problem ce_problem(const float* A, int64_t lda, const float* B, int64_t ldb, float* C, int64_t ldc, int64_t M,
                   int64_t N, int64_t K) {
  return single(A, B, C, M, N, K, lda, ldb, ldc);
}

size_t mm_bytes(const Problem& q, int flags) {
  tilec_mm_cfg cfg = {};
  cfg.flags = flags;
  return workspace_for(q, &cfg);
}

inline bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

int check_ce(const CeCall& c) {
  if (c.dtype < TILEC_DTYPE_F32 || c.dtype > TILEC_DTYPE_BF16) return TILEC_ERR_BAD_ARG;
  if (c.reduction < kReduceNone || c.reduction > kReduceMean) return TILEC_ERR_BAD_ARG;
  if (c.T < 0 || c.V < 1 || c.D < 1 || c.ldx < c.D || c.ldw < c.D) return TILEC_ERR_BAD_ARG;
  if (!c.w || (c.T > 0 && (!c.x || !c.target))) return TILEC_ERR_BAD_ARG;
  const unsigned elem = c.dtype == TILEC_DTYPE_F32 ? 4 : 2;
  if (misaligned(c.x, elem) || misaligned(c.w, elem) || misaligned(c.target, 8)) return TILEC_ERR_BAD_ARG;
  if (c.T >= (int64_t(1) << 30) || c.V >= (int64_t(1) << 30) || c.D >= (int64_t(1) << 30)) return TILEC_ERR_UNSUPPORTED;
  return TILEC_OK;
}

// `grads`: bit 0 the gradient by x, bit 1 by w; 0 = forward.
void plan_ce(const CeCall& c, int grads, const LmInfo& lm, CePlan* p) {
  p->f32 = c.dtype == TILEC_DTYPE_F32;
  p->bf16 = c.dtype == TILEC_DTYPE_BF16;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at = align256(at + bytes);
    return o;
  };
  const bool bwd = grads != 0;
  const int64_t elem = p->f32 ? 4 : 2;
  p->piece = round_up(c.V, 256);
  if (bwd || p->f32) {
    int64_t fit = kCePieceBytes / (elem * c.T) / 256 * 256;
    if (fit < kCePieceMin) fit = kCePieceMin;
    if (p->piece > fit) {
      p->pieces = cdiv(c.V, fit);
      p->piece = round_up(cdiv(c.V, p->pieces), 256);
    }
  }
  p->pieces = cdiv(c.V, p->piece);
  if (p->piece > c.V) p->piece = c.V;
  p->ldp = round_up(p->piece, 8);
  if (!p->f32) {
    p->dp = round_up(c.D, 8);
    // Dropping tokens without a target pays where it can save whole 256-row tiles; the
    // backward pass also needs their rows out of the sum over tokens.
    p->compact = bwd || c.T > 256;
    p->pack_x = p->compact || !rows_aligned16(c.x, c.ldx);
    p->pack_w = !rows_aligned16(c.w, c.ldw);
    p->off_head = take(16);
    if (p->compact) p->off_rows = take(size_t(c.T) * 4);
    if (p->pack_x) p->off_x = take(size_t(c.T) * p->dp * 2);
    if (p->pack_w) p->off_w = take(size_t(c.V) * p->dp * 2);
  }
  if (!bwd) {
    p->nblk = p->f32 ? p->pieces : 2 * cdiv(c.V, 256);
    p->off_part = take(size_t(c.T) * p->nblk * 8);
    p->off_tlogit = take(size_t(c.T) * 4);
    if (c.reduction != kReduceNone) p->off_loss = take(size_t(c.T) * 4);
  }
  if (bwd || p->f32) p->off_p = take(size_t(c.T) * p->ldp * elem);
  if (bwd && !p->f32) {
    p->ldacc = round_up(c.D, 8);
    size_t slabs = 0;
    if (grads & 1) {
      p->dx_slices = f16_slices(c.T, c.D, p->piece, lm, &p->dx_kb);
      if (p->pieces > 1) p->off_acc = take(size_t(c.T) * p->ldacc * 4);
      if (p->dx_slices > 1) slabs = size_t(p->dx_slices) * c.T * p->ldacc * 4;
    }
    if (grads & 2) {
      p->dw_slices = f16_slices(p->piece, c.D, c.T, lm, &p->dw_kb);
      if (p->dw_slices > 1) {
        const size_t b = size_t(p->dw_slices) * p->piece * p->ldacc * 4;
        if (b > slabs) slabs = b;
      }
    }
    if (slabs) p->off_slabs = take(slabs);
    // The gradients lie dense on 16-byte boundaries: whole pieces when D is a multiple of 8.
    size_t odd = 0;
    if ((grads & 1) && p->dx_slices == 1) odd = size_t(c.T) * p->ldacc * 2;
    if ((grads & 2) && p->dw_slices == 1 && size_t(p->piece) * p->ldacc * 2 > odd) odd = size_t(p->piece) * p->ldacc * 2;
    if (odd && c.D % 8 != 0) p->off_odd = take(odd);
  }
  if (p->f32) {
    const float* x = static_cast<const float*>(c.x);
    const float* w = static_cast<const float*>(c.w);
    const int64_t dz = round_up(c.D, 4);
    if (grads & 2) p->off_x = take(size_t(c.T) * dz * 4);
    if ((grads & 1) && p->pieces > 1) p->off_acc = take(size_t(c.T) * c.D * 4);
    const int64_t last = c.V - (p->pieces - 1) * p->piece;
    for (int64_t n : {p->piece, last}) {
      size_t b = mm_bytes(ce_problem(x, c.ldx, w, c.ldw, nullptr, p->ldp, c.T, n, c.D), TILEC_MM_TRANS_B);
      if (b > p->mm_bytes) p->mm_bytes = b;
      if (grads & 1) {
        b = mm_bytes(ce_problem(nullptr, p->ldp, w, c.ldw, nullptr, c.D, c.T, c.D, n), 0);
        if (b > p->mm_bytes) p->mm_bytes = b;
      }
      if (grads & 2) {
        b = mm_bytes(ce_problem(nullptr, p->ldp, nullptr, dz, nullptr, c.D, n, c.D, c.T), TILEC_MM_TRANS_A);
        if (b > p->mm_bytes) p->mm_bytes = b;
      }
    }
    if (p->mm_bytes) p->off_mm = take(p->mm_bytes);
  }
  p->bytes = at;
}

int pack16(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t nrows, int64_t cols, const int* rows,
           const int* count, const int64_t* target, int64_t ignore, void* zero_rows, const DeviceInfo& d,
           cudaStream_t s) {
  int64_t blocks = cdiv(nrows, 8);
  if (blocks > int64_t(d.sms) * 32) blocks = int64_t(d.sms) * 32;
  return launch_k(pack16_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1,
                  static_cast<const unsigned short*>(src), lds, static_cast<unsigned short*>(dst), ldd, nrows, cols,
                  rows, count, rows_aligned16(src, lds) ? 1 : 0, target, ignore,
                  static_cast<unsigned short*>(zero_rows));
}

int run_mm(const Problem& q, int flags, uint8_t* ws, const CePlan& p, cudaStream_t s) {
  tilec_mm_cfg cfg = {};
  cfg.flags = flags;
  return run_problem(q, &cfg, p.mm_bytes ? ws + p.off_mm : nullptr, p.mm_bytes, s);
}

int check_ws(const CePlan& p, void* ws, size_t ws_bytes) {
  return p.bytes > 0 && (!ws || ws_bytes < p.bytes || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
             ? TILEC_ERR_WORKSPACE
             : TILEC_OK;
}

int ce_forward(const CeCall& c, float* loss, float* stats_buf, void* workspace, size_t ws_bytes, cudaStream_t s) {
  DeviceInfo* d = nullptr;
  LmInfo* lm = nullptr;
  TILEC_TRY(lm_device(&d, &lm));
  float2* stats = reinterpret_cast<float2*>(stats_buf);
  float* count_out = stats_buf + 2 * c.T;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (c.T == 0) {
    if (c.reduction == kReduceNone) return TILEC_OK;
    return launch_k(ce_reduce_kernel, dim3(1), dim3(1024), 0, s, 1, static_cast<const float*>(nullptr), int64_t(0),
                    c.target, c.ignore, c.reduction, loss, count_out);
  }
  CePlan p;
  plan_ce(c, 0, *lm, &p);
  TILEC_TRY(check_ws(p, workspace, ws_bytes));
  float2* part = reinterpret_cast<float2*>(ws + p.off_part);
  float* tlogit = reinterpret_cast<float*>(ws + p.off_tlogit);
  float* losses = c.reduction == kReduceNone ? loss : reinterpret_cast<float*>(ws + p.off_loss);
  int* head = reinterpret_cast<int*>(ws + p.off_head);
  int* rows = p.compact ? reinterpret_cast<int*>(ws + p.off_rows) : nullptr;
  const int* count = p.compact ? head : nullptr;
  if (p.f32) {
    float* l = reinterpret_cast<float*>(ws + p.off_p);
    for (int64_t i = 0; i < p.pieces; ++i) {
      const int64_t v0 = i * p.piece, n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
      TILEC_TRY(run_mm(ce_problem(static_cast<const float*>(c.x), c.ldx, static_cast<const float*>(c.w) + v0 * c.ldw,
                                  c.ldw, l, p.ldp, c.T, n, c.D),
                       TILEC_MM_TRANS_B, ws, p, s));
      TILEC_TRY(launch_k(ce_stats_f32_kernel, dim3(static_cast<unsigned>(c.T)), dim3(256), 0, s, 1, l, p.ldp, n, v0,
                         c.target, part, static_cast<int>(p.nblk), static_cast<int>(i), tlogit));
    }
  } else {
    const void* x = c.x;
    const void* w = c.w;
    int64_t ldx = c.ldx, ldw = c.ldw;
    if (p.compact)
      TILEC_TRY(launch_k(ce_select_kernel, dim3(1), dim3(1024), 0, s, 1, c.target, c.T, c.ignore, rows,
                         reinterpret_cast<float*>(head), static_cast<float*>(nullptr),
                         static_cast<const float*>(nullptr), static_cast<const float*>(nullptr), c.reduction, 0));
    if (p.pack_x) {
      TILEC_TRY(pack16(c.x, c.ldx, ws + p.off_x, p.dp, c.T, c.D, rows, count, nullptr, 0, nullptr, *d, s));
      x = ws + p.off_x;
      ldx = p.dp;
    }
    if (p.pack_w) {
      TILEC_TRY(pack16(c.w, c.ldw, ws + p.off_w, p.dp, c.V, c.D, nullptr, nullptr, nullptr, 0, nullptr, *d, s));
      w = ws + p.off_w;
      ldw = p.dp;
    }
    F16Args a = {};
    a.bf16 = p.bf16;
    a.count = count;
    a.rows = rows;
    a.part = part;
    a.tlogit = tlogit;
    a.target = c.target;
    TILEC_TRY((launch_f16<kEpiStats, false, true>(Op16{x, ldx, false}, Op16{w, ldw, false}, c.T, c.V, c.D, a, *lm, s)));
  }
  TILEC_TRY(launch_k(ce_join_kernel, dim3(static_cast<unsigned>(cdiv(c.T, 8))), dim3(256), 0, s, 1, part,
                     static_cast<int>(p.nblk), c.T, c.V, c.target, c.ignore, rows, count, tlogit, stats, losses));
  if (c.reduction == kReduceNone) return TILEC_OK;
  return launch_k(ce_reduce_kernel, dim3(1), dim3(1024), 0, s, 1, losses, c.T, c.target, c.ignore, c.reduction, loss,
                  count_out);
}

int ce_backward_f32(const CeCall& c, const CePlan& p, const float* stats_buf, const float* grad, float* dx, float* dw,
                    uint8_t* ws, const DeviceInfo& d, cudaStream_t s) {
  const float2* stats = reinterpret_cast<const float2*>(stats_buf);
  const float* count = stats_buf + 2 * c.T;
  float* l = reinterpret_cast<float*>(ws + p.off_p);
  float* xz = reinterpret_cast<float*>(ws + p.off_x);
  float* sums = reinterpret_cast<float*>(ws + p.off_acc);
  const int64_t dz = round_up(c.D, 4);
  const unsigned row_blocks = static_cast<unsigned>(c.T < int64_t(d.sms) * 16 ? c.T : int64_t(d.sms) * 16);
  const float* x = static_cast<const float*>(c.x);
  if (dw)
    TILEC_TRY(launch_k(ce_mask_rows_f32_kernel, dim3(row_blocks), dim3(256), 0, s, 1, x, c.ldx, xz, dz, c.T, c.D,
                       c.target, c.ignore));
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
    const float* w = static_cast<const float*>(c.w) + v0 * c.ldw;
    TILEC_TRY(run_mm(ce_problem(x, c.ldx, w, c.ldw, l, p.ldp, c.T, n, c.D), TILEC_MM_TRANS_B, ws, p, s));
    TILEC_TRY(launch_k(ce_prob_f32_kernel, dim3(static_cast<unsigned>(c.T)), dim3(256), 0, s, 1, l, p.ldp, n, v0,
                       c.target, c.ignore, stats, grad, count, c.reduction));
    if (dx) {
      TILEC_TRY(run_mm(ce_problem(l, p.ldp, w, c.ldw, i == 0 ? dx : sums, c.D, c.T, c.D, n), 0, ws, p, s));
      const int last = i == p.pieces - 1;
      if (i > 0 || last)
        TILEC_TRY(launch_k(ce_finish_dx_f32_kernel, dim3(row_blocks), dim3(256), 0, s, 1, dx,
                           static_cast<const float*>(i > 0 ? sums : nullptr), c.T, c.D, c.target, c.ignore, last));
    }
    if (dw)
      TILEC_TRY(run_mm(ce_problem(l, p.ldp, xz, dz, dw + v0 * c.D, c.D, n, c.D, c.T), TILEC_MM_TRANS_A, ws, p, s));
  }
  return TILEC_OK;
}

int ce_backward(const CeCall& c, const float* stats_buf, const float* grad, void* dx, void* dw, void* workspace,
                size_t ws_bytes, cudaStream_t s) {
  const int grads = (dx ? 1 : 0) | (dw ? 2 : 0);
  if (grads == 0) return TILEC_OK;
  DeviceInfo* d = nullptr;
  LmInfo* lm = nullptr;
  TILEC_TRY(lm_device(&d, &lm));
  if (c.T == 0) {
    if (!dw) return TILEC_OK;
    return cudaMemsetAsync(dw, 0, size_t(c.V) * c.D * (c.dtype == TILEC_DTYPE_F32 ? 4 : 2), s) == cudaSuccess
               ? TILEC_OK
               : TILEC_ERR_LAUNCH;
  }
  CePlan p;
  plan_ce(c, grads, *lm, &p);
  TILEC_TRY(check_ws(p, workspace, ws_bytes));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (p.f32)
    return ce_backward_f32(c, p, stats_buf, grad, static_cast<float*>(dx), static_cast<float*>(dw), ws, *d, s);

  float* head = reinterpret_cast<float*>(ws + p.off_head);
  const int* count = reinterpret_cast<const int*>(head);
  float* scale = head + 2;
  int* rows = reinterpret_cast<int*>(ws + p.off_rows);
  TILEC_TRY(launch_k(ce_select_kernel, dim3(1), dim3(1024), 0, s, 1, c.target, c.T, c.ignore, rows, head, scale, grad,
                     stats_buf + 2 * c.T, c.reduction, p.bf16 ? 0 : 1));
  void* xc = ws + p.off_x;
  TILEC_TRY(pack16(c.x, c.ldx, xc, p.dp, c.T, c.D, rows, count, c.target, c.ignore, dx, *d, s));
  const void* w = c.w;
  int64_t ldw = c.ldw;
  if (p.pack_w) {
    TILEC_TRY(pack16(c.w, c.ldw, ws + p.off_w, p.dp, c.V, c.D, nullptr, nullptr, nullptr, 0, nullptr, *d, s));
    w = ws + p.off_w;
    ldw = p.dp;
  }
  // fp16 probabilities are held times 2^15 (the largest magnitude is then 2^15): a token's
  // share 2^-24 of the probability would otherwise already be a subnormal.
  const float pscale = p.bf16 ? 1.f : 32768.f;
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
    const void* wi = static_cast<const unsigned short*>(w) + v0 * ldw;
    void* prob = ws + p.off_p;
    F16Args a = {};
    a.bf16 = p.bf16;
    a.count = count;
    a.rows = rows;
    a.target = c.target;
    a.stats = reinterpret_cast<const float2*>(stats_buf);
    a.grad = c.reduction == kReduceNone ? grad : nullptr;
    a.head = head;
    a.pscale = pscale;
    a.m_alloc = static_cast<int>(c.T);
    a.col0 = static_cast<int>(v0);
    a.out = prob;
    a.ldo = p.ldp;
    TILEC_TRY((launch_f16<kEpiProb, false, true>(Op16{xc, p.dp, false}, Op16{wi, ldw, false}, c.T, n, c.D, a, *lm, s)));
    F16Args g = {};
    g.bf16 = p.bf16;
    g.count = count;
    g.scale = scale;
    g.scale2 = 1.f / pscale;
    float* slabs = reinterpret_cast<float*>(ws + p.off_slabs);
    if (dx) {
      const bool last = i == p.pieces - 1;
      float* acc = reinterpret_cast<float*>(ws + p.off_acc);
      g.rows = rows;
      TILEC_TRY((product16<false, false>(Op16{prob, p.ldp, false}, Op16{wi, ldw, true}, c.T, c.D, n, g, p.dx_slices,
                                         p.dx_kb, p.ldacc, i > 0 ? acc : nullptr, acc, last ? dx : nullptr, c.D, slabs,
                                         ws + p.off_odd, *lm, *d, s)));
    }
    if (dw) {
      g.rows = nullptr;
      g.count_is_k = 1;
      TILEC_TRY((product16<true, false>(Op16{prob, p.ldp, true}, Op16{xc, p.dp, true}, n, c.D, c.T, g, p.dw_slices,
                                        p.dw_kb, p.ldacc, nullptr, nullptr,
                                        static_cast<unsigned short*>(dw) + v0 * c.D, c.D, slabs, ws + p.off_odd, *lm,
                                        *d, s)));
    }
  }
  return TILEC_OK;
}

CeCall ce_call(const void* x, const void* w, const int64_t* target, int32_t dtype, int64_t T, int64_t V, int64_t D,
               int64_t ldx, int64_t ldw, int64_t ignore, int32_t reduction) {
  return CeCall{x, w, target, dtype, T, V, D, ldx, ldw, ignore, reduction};
}

// ---------------------------------------------------------------- 4-bit weights
// Bytes of expanded weights held at a time where x has many rows.
constexpr int64_t kW4ExpandBytes = int64_t(256) << 20;

struct W4Call {
  const void* x;
  int dtype;
  int64_t M, ldx;
  const void* weight;
  int sdt;
  int64_t N, K, group;
  const void* bias;
  void* out;
  int64_t ldo;
};

// Shared memory of w4_stream_kernel without x.
template <int NT, int XT>
int64_t w4_stream_fixed_nt(int gpb, bool wide) {
  return gpb == 4   ? (wide ? W4StreamCfg<NT, 4, true, XT>::kFixed : W4StreamCfg<NT, 4, false, XT>::kFixed)
         : gpb == 2 ? (wide ? W4StreamCfg<NT, 2, true, XT>::kFixed : W4StreamCfg<NT, 2, false, XT>::kFixed)
                    : (wide ? W4StreamCfg<NT, 1, true, XT>::kFixed : W4StreamCfg<NT, 1, false, XT>::kFixed);
}
int64_t w4_stream_fixed(int nt, int gpb, bool wide, int xt) {
  if (xt == 0) return w4_stream_fixed_nt<1, 0>(gpb, wide);
  if (xt == kW4Terms) return nt == 1 ? w4_stream_fixed_nt<1, kW4Terms>(gpb, wide) : w4_stream_fixed_nt<3, kW4Terms>(gpb, wide);
  return nt == 1 ? w4_stream_fixed_nt<1, TILEC_DTYPE_BF16>(gpb, wide) : w4_stream_fixed_nt<2, TILEC_DTYPE_BF16>(gpb, wide);
}

struct W4Plan {
  bool stream = false;   // w4_stream_kernel
  int xt = 0;            // ... how x enters it: digits, its 16-bit type or three terms
  bool tc = false;       // w4_tc_kernel; otherwise expanded weights and a plain product
  bool pack_x = false;   // x is copied to aligned rows first (expanded weights)
  int nt = 1, cols = 1, splits = 1, slab = 1, per_cta = 0, ctas = 0;
  bool polling = false;  // w4_stream_kernel's waits, see W4StreamArgs
  int64_t blocks = 0, kp = 0, piece = 0;
  int slices = 1, kb = 0;
  int64_t ldslab = 0;
  size_t off_x = 0, off_w = 0, off_slabs = 0, off_odd = 0, off_mm = 0, mm_bytes = 0, bytes = 0;
};

int check_w4(const W4Call& c) {
  if (c.dtype < TILEC_DTYPE_F32 || c.dtype > TILEC_DTYPE_BF16 || c.sdt < TILEC_DTYPE_F32 || c.sdt > TILEC_DTYPE_BF16)
    return TILEC_ERR_BAD_ARG;
  if (c.M < 0 || c.N < 0 || c.K < 1 || c.ldx < c.K) return TILEC_ERR_BAD_ARG;
  if (c.group != 32 && c.group != 64 && (c.group < 128 || c.group % 128 != 0)) return TILEC_ERR_BAD_ARG;
  if (c.M >= (int64_t(1) << 30) || c.N >= (int64_t(1) << 30) || c.K >= (int64_t(1) << 30) ||
      c.group >= (int64_t(1) << 31))
    return TILEC_ERR_UNSUPPORTED;
  return TILEC_OK;
}

int check_w4_pointers(const W4Call& c) {
  if (c.M == 0 || c.N == 0) return TILEC_OK;
  if (!c.x || !c.weight || !c.out || c.ldo < c.N) return TILEC_ERR_BAD_ARG;
  const unsigned elem = c.dtype == TILEC_DTYPE_F32 ? 4 : 2;
  if (misaligned(c.weight, 16) || misaligned(c.x, elem) || misaligned(c.out, elem) || misaligned(c.bias, elem))
    return TILEC_ERR_BAD_ARG;
  return TILEC_OK;
}

// How many rows of x run where: one of 16-bit x in digits on w4_stream_kernel; up to 16 there too,
// as they are; up to 8 of fp32 x there as well, in three bf16 terms (three columns a row, which
// NT = 3 tiles of 8 hold); up to 256 of 16-bit x whose type the scales share on w4_tc_kernel, 128
// at a time (8192 x 8192: 128 rows 35 to 39 us, twice that for 256; expanded first, either takes
// 89); for the rest W is expanded once into the workspace and multiplied on the tcgen05 kernels
// (fp32: 3xTF32).
constexpr int64_t kW4Max16 = 16;    // rows of 16-bit x
constexpr int64_t kW4Max32 = 8;     // rows of fp32 x

void plan_w4(const W4Call& c, const DeviceInfo& d, const LmInfo& lm, W4Plan* p) {
  const bool f32 = c.dtype == TILEC_DTYPE_F32;
  p->blocks = cdiv(c.K, kW4Block);
  p->kp = p->blocks * kW4Block;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at = align256(at + bytes);
    return o;
  };
  const int gpb = c.group == 32 ? 4 : c.group == 64 ? 2 : 1;
  const bool wide = c.sdt == TILEC_DTYPE_F32;
  const bool digits = !f32 && c.M == 1, terms = f32 && c.M <= kW4Max32;
  // Nine to 16 rows: each further slab of x costs w4_stream_kernel some 6 us, w4_tc_kernel is the
  // slower the larger the weight (4096 x 4096, 16 rows in two slabs: 18.0 against 11.3 us;
  // 8192 x 8192, 13 in two: 22.8 against 25.6, 16 in three: 28.0 against 25.6; 28672 x 8192, 16
  // in three: 52 against 82).
  bool in16 = !f32 && c.M <= kW4Max16;
  if (in16 && c.M > 8 && c.sdt == c.dtype) {
    const int64_t slabs =
        cdiv(w4_slab16_bytes(p->blocks, c.M), kW4MaxSmem - w4_stream_fixed(2, gpb, wide, c.dtype));
    in16 = c.N * p->kp >= (slabs - 1) << 26;
  }
  if (digits || in16 || terms) {
    p->stream = true;
    p->polling = d.short_waits;
    p->xt = digits ? 0 : terms ? kW4Terms : c.dtype;
    p->cols = static_cast<int>(digits ? kW4Digits : terms ? kW4Terms * c.M : c.M);
    p->nt = terms ? (c.M <= 2 ? 1 : 3) : p->cols <= 8 ? 1 : 2;
    // One CTA per SM.  With fewer 16-row tiles than SMs, a cluster of CTAs shares each tile's K.
    const int64_t tiles = cdiv(c.N, 16);
    int64_t splits = d.sms / tiles;
    if (splits > 8) splits = 8;
    if (splits > p->blocks / 4) splits = p->blocks / 4;
    if (splits < 1) splits = 1;
    p->per_cta = static_cast<int>(cdiv(p->blocks, splits));
    p->splits = static_cast<int>(cdiv(p->blocks, p->per_cta));
    const int64_t clusters = d.sms / p->splits;
    p->ctas = static_cast<int>((tiles < clusters ? tiles : clusters) * p->splits);
    const int64_t room = kW4MaxSmem - w4_stream_fixed(p->nt, gpb, wide, p->xt);
    auto slab_bytes = [&](int64_t n) { return digits ? w4_slab_bytes(n, gpb) : w4_slab16_bytes(n, p->cols); };
    int64_t slab = p->per_cta;
    while (slab > 1 && slab_bytes(slab) > room) --slab;
    p->slab = static_cast<int>(cdiv(p->per_cta, cdiv(p->per_cta, slab)));  // slabs of one size
  } else if (!f32 && c.M <= 2 * W4TcCfg<1>::kMaxCols && c.sdt == c.dtype) {
    p->tc = true;
    p->pack_x = !rows_aligned16(c.x, c.ldx);
    if (p->pack_x) p->off_x = take(size_t(c.M) * p->kp * 2);
    // K splits: waves of one CTA per SM, each split's share of K, and about a microsecond's
    // worth (4 blocks) of start-up per CTA and of slab traffic per split.
    const int64_t tiles = cdiv(c.N, W4TcCfg<1>::kRows);
    double best = 0;
    for (int sp = 1; sp <= 8 && sp * 4 <= p->blocks + 3; ++sp) {
      const double cost = double(cdiv(tiles * sp, d.sms)) * (double(cdiv(p->blocks, sp)) + 8.0) + 2.0 * (sp - 1);
      if (sp == 1 || cost < best) {
        best = cost;
        p->splits = sp;
      }
    }
    p->per_cta = static_cast<int>(round_up(cdiv(p->blocks, p->splits), 2));
    p->splits = static_cast<int>(cdiv(p->blocks, p->per_cta));
    p->ldslab = round_up(c.N, 8);
    if (p->splits > 1)
      p->off_slabs =
          take(size_t(p->splits) * (c.M < W4TcCfg<1>::kMaxCols ? c.M : W4TcCfg<1>::kMaxCols) * p->ldslab * 4);
  } else {
    int64_t piece = kW4ExpandBytes / (p->kp * (f32 ? 4 : 2)) / 256 * 256;
    if (piece < 256) piece = 256;
    p->piece = c.N < piece ? c.N : piece;
    p->off_w = take(size_t(p->piece) * p->kp * (f32 ? 4 : 2));
    if (f32) {
      const int64_t last = c.N - (cdiv(c.N, p->piece) - 1) * p->piece;
      for (int64_t n : {p->piece, last}) {
        Problem q = single(static_cast<const float*>(c.x), nullptr, static_cast<float*>(c.out), c.M, n, c.K, c.ldx,
                           p->kp, c.ldo > 0 ? c.ldo : c.N);
        const size_t b = mm_bytes(q, TILEC_MM_TRANS_B);
        if (b > p->mm_bytes) p->mm_bytes = b;
      }
      if (p->mm_bytes) p->off_mm = take(p->mm_bytes);
    } else {
      p->pack_x = !rows_aligned16(c.x, c.ldx);
      if (p->pack_x) p->off_x = take(size_t(c.M) * p->kp * 2);
      p->slices = f16_slices(c.M, p->piece, c.K, lm, &p->kb);
      p->ldslab = round_up(p->piece, 8);
      if (p->slices > 1) p->off_slabs = take(size_t(p->slices) * c.M * p->ldslab * 4);
      else if (odd_rows(c.out, c.ldo, c.N)) p->off_odd = take(size_t(c.M) * p->ldslab * 2);
    }
  }
  p->bytes = at;
}

template <int NT, int GPB, int SC, int XT>
int launch_w4_stream(const W4Args& w, const W4Plan& p, cudaStream_t s) {
  W4StreamArgs a;
  a.w = w;
  a.row_tiles = static_cast<int>(cdiv(w.N, 16));
  a.per_cta = p.per_cta;
  a.slab = p.slab;
  a.polling = p.polling;
  using Cfg = W4StreamCfg<NT, GPB, SC == 0, XT>;
  const size_t smem =
      size_t(Cfg::kFixed + (XT != 0 ? w4_slab16_bytes(p.slab, w.cols) : w4_slab_bytes(p.slab, GPB)));
  if (int64_t(smem) > kW4MaxSmem) return TILEC_ERR_UNSUPPORTED;
  return launch_k(w4_stream_kernel<NT, GPB, SC, XT>, dim3(static_cast<unsigned>(p.ctas)), dim3(Cfg::kThreads), smem, s,
                  w.splits, a);
}

// The kernel's variants: by columns, groups per block, type of x and scales.
template <int GPB, bool WIDE>
int launch_w4(const W4Args& a, const W4Plan& p, cudaStream_t s) {
  constexpr int SC = WIDE ? 0 : 1;
  if (p.xt == kW4Terms)
    return p.nt == 1 ? launch_w4_stream<1, GPB, SC, kW4Terms>(a, p, s) : launch_w4_stream<3, GPB, SC, kW4Terms>(a, p, s);
  if (p.xt == TILEC_DTYPE_BF16)
    return p.nt == 1 ? launch_w4_stream<1, GPB, SC, TILEC_DTYPE_BF16>(a, p, s)
                     : launch_w4_stream<2, GPB, SC, TILEC_DTYPE_BF16>(a, p, s);
  if (p.xt == TILEC_DTYPE_F16)
    return p.nt == 1 ? launch_w4_stream<1, GPB, SC, TILEC_DTYPE_F16>(a, p, s)
                     : launch_w4_stream<2, GPB, SC, TILEC_DTYPE_F16>(a, p, s);
  if constexpr (WIDE)
    return launch_w4_stream<1, GPB, TILEC_DTYPE_F32, 0>(a, p, s);
  else
    return a.scale_bf16 ? launch_w4_stream<1, GPB, TILEC_DTYPE_BF16, 0>(a, p, s)
                        : launch_w4_stream<1, GPB, TILEC_DTYPE_F16, 0>(a, p, s);
}

template <bool WIDE>
int launch_w4(const W4Args& a, const W4Plan& p, int gpb, cudaStream_t s) {
  return gpb == 4   ? launch_w4<4, WIDE>(a, p, s)
         : gpb == 2 ? launch_w4<2, WIDE>(a, p, s)
                    : launch_w4<1, WIDE>(a, p, s);
}

template <bool BF16, int GPB>
int launch_w4_tc(const W4Args& w, const W4Plan& p, const CUtensorMap& tm, float* slabs, cudaStream_t s) {
  W4TcArgs a;
  a.w = w;
  a.n_cols = static_cast<int>(round_up(w.M, 16));
  a.per_cta = p.per_cta;
  a.slabs = slabs;
  a.lds = p.ldslab;
  return launch_k(w4_tc_kernel<BF16, GPB>, dim3(static_cast<unsigned>(cdiv(w.N, W4TcCfg<GPB>::kRows) * w.splits)),
                  dim3(W4TcCfg<GPB>::kThreads), W4TcCfg<GPB>::kSmemBytes, s, 1, tm, a);
}

int run_w4_tc(const W4Call& c, const W4Plan& p, W4Args a, int gpb, uint8_t* ws, const DeviceInfo& d, cudaStream_t s) {
  const bool bf16 = c.dtype == TILEC_DTYPE_BF16;
  const void* x = c.x;
  int64_t ldx = c.ldx;
  if (p.pack_x) {
    TILEC_TRY(pack16(c.x, c.ldx, ws + p.off_x, p.kp, c.M, c.K, nullptr, nullptr, nullptr, 0, nullptr, d, s));
    x = ws + p.off_x;
    ldx = p.kp;
  }
  float* slabs = reinterpret_cast<float*>(ws + p.off_slabs);
  constexpr int64_t kStep = W4TcCfg<1>::kMaxCols;
  for (int64_t m0 = 0; m0 < c.M; m0 += kStep) {
    const int64_t m = c.M - m0 < kStep ? c.M - m0 : kStep;
    CUtensorMap tm;
    TILEC_TRY(encode16(&tm, static_cast<const unsigned short*>(x) + m0 * ldx, c.K, m, ldx,
                       static_cast<int>(round_up(m, 16)), bf16));
    unsigned short* out = static_cast<unsigned short*>(c.out) + m0 * c.ldo;
    a.M = static_cast<int>(m);
    a.out = out;
    if (bf16)
      TILEC_TRY((gpb == 4   ? launch_w4_tc<true, 4>(a, p, tm, slabs, s)
                 : gpb == 2 ? launch_w4_tc<true, 2>(a, p, tm, slabs, s)
                            : launch_w4_tc<true, 1>(a, p, tm, slabs, s)));
    else
      TILEC_TRY((gpb == 4   ? launch_w4_tc<false, 4>(a, p, tm, slabs, s)
                 : gpb == 2 ? launch_w4_tc<false, 2>(a, p, tm, slabs, s)
                            : launch_w4_tc<false, 1>(a, p, tm, slabs, s)));
    if (p.splits == 1) continue;
    int64_t blocks = cdiv(m * cdiv(c.N, 8), 256);
    if (blocks > int64_t(d.sms) * 8) blocks = int64_t(d.sms) * 8;
    TILEC_TRY(launch_k(f16_join_slabs_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1,
                       static_cast<const float*>(slabs), p.splits, m * p.ldslab, p.ldslab,
                       static_cast<const float*>(nullptr), static_cast<float*>(nullptr), out, c.ldo, m, c.N,
                       static_cast<const int*>(nullptr), static_cast<const int*>(nullptr),
                       static_cast<const float*>(nullptr), 1.f, c.bias, bf16 ? 1 : 0,
                       odd_rows(out, c.ldo, c.N) ? 0 : 1));
  }
  return TILEC_OK;
}

int run_w4(const W4Call& c, void* workspace, size_t ws_bytes, cudaStream_t s) {
  DeviceInfo* d = nullptr;
  LmInfo* lm = nullptr;
  TILEC_TRY(lm_device(&d, &lm));
  W4Plan p;
  plan_w4(c, *d, *lm, &p);
  if (p.bytes > 0 && (!workspace || ws_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
    return TILEC_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool f32 = c.dtype == TILEC_DTYPE_F32;
  W4Args a = {};
  a.data = static_cast<const uint8_t*>(c.weight);
  a.wide = c.sdt == TILEC_DTYPE_F32;
  a.scale_bf16 = c.sdt == TILEC_DTYPE_BF16;
  a.N = static_cast<int>(c.N);
  a.K = static_cast<int>(c.K);
  a.blocks = static_cast<int>(p.blocks);
  const int gpb = c.group == 32 ? 4 : c.group == 64 ? 2 : 1;
  if (p.stream || p.tc) {
    a.x = c.x;
    a.ldx = c.ldx;
    a.dtype = c.dtype;
    a.M = static_cast<int>(c.M);
    a.cols = p.cols;
    a.vec_x = aligned16(c.x) && c.ldx % (f32 ? 4 : 8) == 0;
    a.out = c.out;
    a.ldo = c.ldo;
    a.bias = c.bias;
    a.splits = p.splits;
    if (p.tc) return run_w4_tc(c, p, a, gpb, ws, *d, s);
    return a.wide ? launch_w4<true>(a, p, gpb, s) : launch_w4<false>(a, p, gpb, s);
  }
  const void* x = c.x;
  int64_t ldx = c.ldx;
  if (p.pack_x) {
    TILEC_TRY(pack16(c.x, c.ldx, ws + p.off_x, p.kp, c.M, c.K, nullptr, nullptr, nullptr, 0, nullptr, *d, s));
    x = ws + p.off_x;
    ldx = p.kp;
  }
  void* wd = ws + p.off_w;
  const int64_t elem = f32 ? 4 : 2;
  for (int64_t n0 = 0; n0 < c.N; n0 += p.piece) {
    const int64_t n = c.N - n0 < p.piece ? c.N - n0 : p.piece;
    int64_t blocks = cdiv(n * p.blocks * 16, 256);
    if (blocks > int64_t(d->sms) * 16) blocks = int64_t(d->sms) * 16;
    TILEC_TRY(launch_k(w4_expand_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1, a,
                       static_cast<int>(n0), static_cast<int>(n), gpb, c.dtype, wd, p.kp));
    uint8_t* out = static_cast<uint8_t*>(c.out) + n0 * elem;
    const uint8_t* bias = c.bias ? static_cast<const uint8_t*>(c.bias) + n0 * elem : nullptr;
    if (f32) {
      Problem q = single(static_cast<const float*>(x), static_cast<const float*>(wd), reinterpret_cast<float*>(out),
                         c.M, n, c.K, ldx, p.kp, c.ldo);
      q.bias = reinterpret_cast<const float*>(bias);
      tilec_mm_cfg cfg = {};
      cfg.flags = TILEC_MM_TRANS_B;
      TILEC_TRY(run_problem(q, &cfg, p.mm_bytes ? ws + p.off_mm : nullptr, p.mm_bytes, s));
    } else {
      F16Args f = {};
      f.bf16 = c.dtype == TILEC_DTYPE_BF16;
      f.scale2 = 1.f;
      f.bias = bias;
      TILEC_TRY((product16<false, true>(Op16{x, ldx, false}, Op16{wd, p.kp, false}, c.M, n, c.K, f, p.slices, p.kb,
                                        p.ldslab, nullptr, nullptr, out, c.ldo,
                                        reinterpret_cast<float*>(ws + p.off_slabs), ws + p.off_odd, *lm, *d, s)));
    }
  }
  return TILEC_OK;
}

}  // namespace
}  // namespace tilec

extern "C" {

size_t tilec_linear_ce_workspace_bytes(const void* x, const void* w, int32_t dtype, int64_t T, int64_t V, int64_t D,
                                       int64_t ldx, int64_t ldw, int32_t reduction, int32_t grads) {
  static const int64_t kSome = 0;
  const CeCall c = ce_call(x ? x : reinterpret_cast<const void*>(256), w ? w : reinterpret_cast<const void*>(256),
                           &kSome, dtype, T, V, D, ldx, ldw, 0, reduction);
  if (check_ce(c) || T == 0 || grads < 0 || grads > 3) return 0;
  DeviceInfo* d = nullptr;
  LmInfo* lm = nullptr;
  if (lm_device(&d, &lm)) return 0;
  CePlan p;
  plan_ce(c, grads, *lm, &p);
  return p.bytes;
}

int tilec_linear_ce_forward(const void* x, const void* w, const int64_t* target, int32_t dtype, int64_t T, int64_t V,
                            int64_t D, int64_t ldx, int64_t ldw, int64_t ignore_index, int32_t reduction, float* loss,
                            float* stats, void* workspace, size_t ws_bytes, void* stream) {
  const CeCall c = ce_call(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction);
  const int rc = check_ce(c);
  if (rc) return rc;
  if (!stats || (!loss && (T > 0 || reduction != kReduceNone))) return TILEC_ERR_BAD_ARG;
  if (misaligned(stats, 8) || misaligned(loss, 4)) return TILEC_ERR_BAD_ARG;
  return ce_forward(c, loss, stats, workspace, ws_bytes, static_cast<cudaStream_t>(stream));
}

int tilec_linear_ce_backward(const void* x, const void* w, const int64_t* target, int32_t dtype, int64_t T, int64_t V,
                             int64_t D, int64_t ldx, int64_t ldw, int64_t ignore_index, int32_t reduction,
                             const float* stats, const float* grad, void* dx, void* dw, void* workspace,
                             size_t ws_bytes, void* stream) {
  const CeCall c = ce_call(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction);
  const int rc = check_ce(c);
  if (rc) return rc;
  if (!stats || (!grad && (T > 0 || reduction != kReduceNone))) return TILEC_ERR_BAD_ARG;
  if (!aligned16(dx) || !aligned16(dw) || misaligned(stats, 8) || misaligned(grad, 4)) return TILEC_ERR_BAD_ARG;
  return ce_backward(c, stats, grad, dx, dw, workspace, ws_bytes, static_cast<cudaStream_t>(stream));
}

size_t tilec_mm_w4_workspace_bytes(const void* x, int32_t dtype, int64_t M, int64_t ldx, int32_t scale_dtype,
                                   int64_t N, int64_t K, int64_t group, const void* out, int64_t ldo) {
  W4Call c = {};
  c.sdt = scale_dtype;
  c.x = x ? x : reinterpret_cast<const void*>(256);
  c.dtype = dtype;
  c.M = M;
  c.ldx = ldx;
  c.N = N;
  c.K = K;
  c.group = group;
  c.out = const_cast<void*>(out);
  c.ldo = ldo;
  if (check_w4(c) || M == 0 || N == 0 || ldo < N) return 0;
  DeviceInfo* d = nullptr;
  LmInfo* lm = nullptr;
  if (lm_device(&d, &lm)) return 0;
  W4Plan p;
  plan_w4(c, *d, *lm, &p);
  return p.bytes;
}

int tilec_mm_w4(const void* x, int32_t dtype, int64_t M, int64_t ldx, const void* weight,
                int32_t scale_dtype, int64_t N, int64_t K, int64_t group, const void* bias, void* out, int64_t ldo,
                void* workspace, size_t ws_bytes, void* stream) {
  const W4Call c{x, dtype, M, ldx, weight, scale_dtype, N, K, group, bias, out, ldo};
  int rc = check_w4(c);
  if (rc) return rc;
  rc = check_w4_pointers(c);
  if (rc || M == 0 || N == 0) return rc;
  return run_w4(c, workspace, ws_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
