// linear_ce.cuh -- the kernels around the products of the fused linear cross entropy:
// row selection and packing, the softmax statistics' join, the loss, and the fp32 path's
// element-wise passes.
//
//   logit_tv = x_t . w_v      loss_t = log sum_v exp(logit_tv) - logit_t,y(t)
//   d loss_t / d logit_tv = softmax_tv - [v = y(t)]
//
// All of them are bound by memory or, at a few rows, by latency; each is a few percent of
// the products it serves.  Softmax statistics live in the log2 domain: a row's pair (m, s)
// stands for sum_v exp(logit) = s * 2^m with m = max(logit) * log2(e), sums in fp32.
#pragma once

#include "common.cuh"
#include "tc2_f16.cuh"

namespace tilec {

enum : int { kReduceNone = 0, kReduceSum = 1, kReduceMean = 2 };

// Joins two partial softmax sums.
__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float ref = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * ex2(a.x - ref) + b.y * ex2(b.x - ref));
}

// One block.  rows[0 .. n) = the tokens that have a target, in order, n to head_int[0].
// Backward only (scale != nullptr): *scale = G and head[1] = 1 / G, where the gradients
// are G times what the products see: the loss's gradient (over the count for the mean), so
// that the probabilities stay in [-1, 1] whatever it is; per-token gradients are part of
// the probabilities, in fp16 divided by their largest magnitude.
__global__ void __launch_bounds__(1024) ce_select_kernel(const int64_t* __restrict__ target, int64_t T, int64_t ignore,
                                                         int* rows, float* head, float* scale, const float* grad,
                                                         const float* count, int reduction, int f16) {
  __shared__ int warp_sum[32];
  __shared__ float warp_max[32];
  __shared__ int base;
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) base = 0;
  float gmax = 0.f;
  const bool per_token = scale != nullptr && reduction == kReduceNone;
  __syncthreads();
  for (int64_t t0 = 0; t0 < T; t0 += 1024) {
    const int64_t t = t0 + tid;
    const bool live = t < T && target[t] != ignore;
    if (live && per_token) {
      const float a = fabsf(grad[t]);
      gmax = a > gmax || a != a ? a : gmax;  // a NaN stays
    }
    const unsigned ballot = __ballot_sync(0xffffffffu, live);
    if (lane == 0) warp_sum[warp] = __popc(ballot);
    __syncthreads();
    int before = base;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (live) rows[before + __popc(ballot & ((1u << lane) - 1u))] = static_cast<int>(t);
    __syncthreads();
    if (tid == 1023) base = before + warp_sum[31];
    __syncthreads();
  }
  if (tid == 0) reinterpret_cast<int*>(head)[0] = base;
  if (scale == nullptr) return;
  if (!per_token) {
    if (tid == 0) {
      // No token has a target: sums are empty, and 1 / 0 (or an infinite grad) times their
      // zeros would be NaN.
      *scale = base == 0 ? 0.f : reduction == kReduceMean ? grad[0] / count[0] : grad[0];
      head[1] = 1.f;
    }
    return;
  }
  float g = 1.f;
  if (f16) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, gmax, o);
      gmax = other > gmax || other != other ? other : gmax;
    }
    if (lane == 0) warp_max[warp] = gmax;
    __syncthreads();
    g = 0.f;
    for (int w = 0; w < 32; ++w) g = warp_max[w] > g || warp_max[w] != warp_max[w] ? warp_max[w] : g;
    // A power of two, so that dividing and multiplying back round nothing.
    if (g > 0.f && g < INFINITY) {
      int ex = 0;
      frexpf(g, &ex);
      g = ldexpf(1.f, max(-126, min(ex, 126)));  // with 1 / g a number too
    } else {
      g = 1.f;
    }
  }
  if (tid == 0) {
    *scale = g;
    head[1] = 1.f / g;
  }
}

// 16-bit rows to an aligned buffer: dst row r = src row rows[r] (or r when rows == nullptr),
// for r < *count (or nrows); rows from there to the end of the last 256-row tile are zeroed,
// so that the gradient product can run over whole blocks of them.  `zero_rows` (the gradient
// by x, or nullptr): tokens without a target get zeros there, their products never run.
// A warp per row, 8 elements a lane; sources that are not 16-byte aligned are read by
// element.
__global__ void __launch_bounds__(256) pack16_kernel(const unsigned short* __restrict__ src, int64_t lds,
                                                     unsigned short* __restrict__ dst, int64_t ldd, int64_t nrows,
                                                     int64_t cols, const int* __restrict__ rows,
                                                     const int* __restrict__ count, int vec,
                                                     const int64_t* __restrict__ target, int64_t ignore,
                                                     unsigned short* zero_rows) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t n = count != nullptr ? *count : nrows;
  int64_t n_zero = (n + 255) / 256 * 256;
  if (n_zero > nrows) n_zero = nrows;
  const int64_t warps = int64_t(gridDim.x) * (blockDim.x >> 5);
  for (int64_t r = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); r < nrows; r += warps) {
    if (zero_rows != nullptr && target[r] == ignore)
      for (int64_t c = lane; c < cols; c += 32) zero_rows[r * cols + c] = 0;
    if (r >= n_zero) continue;
    const bool live = r < n;
    const unsigned short* s = src + (live ? (rows != nullptr ? int64_t(rows[r]) : r) : 0) * lds;
    unsigned short* d = dst + r * ldd;
    for (int64_t c = 8 * lane; c < cols; c += 256) {
      uint4 h = make_uint4(0, 0, 0, 0);
      if (live) {
        if (vec && c + 8 <= cols) {
          h = *reinterpret_cast<const uint4*>(s + c);
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
          if (c + 8 <= cols) {
            // Aligned 4-byte words, shifted into place: each holds an element of the row, so
            // none lies on another page.
            const uintptr_t at = reinterpret_cast<uintptr_t>(s + c);
            const uint32_t* v = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
            const unsigned shift = (at & 2) * 8;
            uint32_t lo = v[0];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t hi = j < 3 || shift ? v[j + 1] : 0u;
              w[j] = __funnelshift_r(lo, hi, shift);
              lo = hi;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c + j < cols) w[j >> 1] |= uint32_t(s[c + j]) << (16 * (j & 1));
          }
          h = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      *reinterpret_cast<uint4*>(d + c) = h;
    }
  }
}

// A warp per product row: joins the row's partial sums and writes, by token, the statistics
// and the loss.  Tokens without a target get a loss of zero from the warp that owns their
// position among all tokens.  A target outside [0, V) is neither a class nor ignored: the
// row's loss and statistics become NaN (its gradients follow) and the status word says so.
__global__ void __launch_bounds__(256) ce_join_kernel(const float2* __restrict__ part, int nblk, int64_t T, int64_t V,
                                                      const int64_t* __restrict__ target, int64_t ignore,
                                                      const int* __restrict__ rows, const int* __restrict__ count,
                                                      const float* __restrict__ tlogit, float2* __restrict__ stats,
                                                      float* __restrict__ loss) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t r = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (r >= T) return;
  if (target[r] == ignore && lane == 0) {
    loss[r] = 0.f;
    stats[r] = make_float2(0.f, 1.f);
  }
  int64_t tok = r;
  if (rows != nullptr) {
    if (r >= *count) return;
    tok = rows[r];
  }
  const int64_t y = target[tok];
  if (y == ignore) return;
  const float2* row = part + r * nblk;
  float2 st = make_float2(-INFINITY, 0.f);
  for (int i = lane; i < nblk; i += 32) st = join_stats(st, row[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 b = make_float2(__shfl_xor_sync(0xffffffffu, st.x, o), __shfl_xor_sync(0xffffffffu, st.y, o));
    st = join_stats(st, b);
  }
  if (lane != 0) return;
  if (y < 0 || y >= V) {
    const float nan = __int_as_float(0x7fc00000);
    record_status(TILEC_DEV_BAD_INDEX);
    stats[tok] = make_float2(nan, nan);
    loss[tok] = nan;
    return;
  }
  stats[tok] = st;
  loss[tok] = kLn2 * (log2f(st.y) + (st.x - tlogit[tok]));
}

// One block: out = sum (or mean over the tokens with a target) of the losses, in fixed order
// and 64 bits; count[0] = how many have a target.
__global__ void __launch_bounds__(1024) ce_reduce_kernel(const float* __restrict__ loss, int64_t T,
                                                         const int64_t* __restrict__ target, int64_t ignore,
                                                         int reduction, float* out, float* count) {
  __shared__ double s_sum[32];
  __shared__ int s_n[32];
  pdl_wait();
  double sum = 0.0;
  int n = 0;
  for (int64_t t = threadIdx.x; t < T; t += 1024) {
    sum += double(loss[t]);
    n += target[t] != ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_n[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0.0;
  n = 0;
  for (int w = 0; w < 32; ++w) {
    sum += s_sum[w];
    n += s_n[w];
  }
  count[0] = float(n);
  if (reduction == kReduceSum) out[0] = float(sum);
  if (reduction == kReduceMean) out[0] = float(sum / double(n));
}

// out (16-bit, rows scattered by `rows`) or acc (fp32) = the K slices' slabs, added in order,
// plus the earlier sums.  A thread per 8 columns.
__global__ void __launch_bounds__(256) f16_join_slabs_kernel(const float* __restrict__ slabs, int slices, int64_t slab,
                                                             int64_t lds, const float* acc_in, float* acc_out,
                                                             unsigned short* out, int64_t ldo, int64_t M, int64_t N,
                                                             const int* __restrict__ count,
                                                             const int* __restrict__ rows, const float* scale,
                                                             float scale2, const void* bias, int bf16, int vec_out) {
  pdl_wait();
  pdl_launch_dependents();
  if (count != nullptr) M = *count;
  const int64_t pieces = (N + 7) / 8, total = M * pieces;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / pieces, c = (i - r * pieces) * 8;
    float x[8] = {};
    auto add = [&](const float* p) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
      x[4] += b.x; x[5] += b.y; x[6] += b.z; x[7] += b.w;
    };
    if (acc_in != nullptr) add(acc_in + r * lds + c);
    for (int s = 0; s < slices; ++s) add(slabs + s * slab + r * lds + c);
    if (out == nullptr) {
      float4* d = reinterpret_cast<float4*>(acc_out + r * lds + c);
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
      continue;
    }
    const float f = (scale != nullptr ? *scale : 1.f) * scale2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] *= f;
      if (bias != nullptr && c + j < N) x[j] += load_16(bias, c + j, bf16);
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_16x2(x[2 * j], x[2 * j + 1], bf16);
    unsigned short* d = out + (rows != nullptr ? int64_t(rows[r]) : r) * ldo + c;
    if (vec_out && c + 8 <= N) {
      *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < N) d[j] = static_cast<unsigned short>(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Rows of `src` (row stride lds) to rows of `dst` that 16-byte stores cannot take, dst row
// rows[r] (or r).  The product kernel stores whole 8-column pieces; storing odd rows from there
// cost 155 us for the gradient of a 30011 x 777 weight, through this copy it is 76 (50 + 26).  Dense rows
// (rows == nullptr, ldd == cols) go out as one run, 16 bytes a thread; others by element.
__global__ void __launch_bounds__(256) unpad16_kernel(const unsigned short* __restrict__ src, int64_t lds,
                                                      unsigned short* __restrict__ dst, int64_t ldd, int64_t nrows,
                                                      int cols, const int* __restrict__ count,
                                                      const int* __restrict__ rows, int dense) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t n = count != nullptr ? *count : nrows;
  const int64_t threads = int64_t(gridDim.x) * 256, self = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (dense) {
    const int64_t total = n * cols;
    for (int64_t i = self * 8; i < total; i += threads * 8) {
      int64_t r = i / cols;
      int c = static_cast<int>(i - r * cols);
      uint32_t w[4] = {0, 0, 0, 0};
      const int m = total - i < 8 ? static_cast<int>(total - i) : 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < m) w[j >> 1] |= uint32_t(src[r * lds + c]) << (16 * (j & 1));
        if (++c == cols) {
          c = 0;
          ++r;
        }
      }
      if (m == 8) {
        *reinterpret_cast<uint4*>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < m) dst[i + j] = static_cast<unsigned short>(w[j >> 1] >> (16 * (j & 1)));
      }
    }
    return;
  }
  for (int64_t i = self; i < n * cols; i += threads) {
    const int64_t r = i / cols;
    dst[(rows != nullptr ? int64_t(rows[r]) : r) * ldd + (i - r * cols)] = src[r * lds + (i - r * cols)];
  }
}

// ---------------------------------------------------------------- fp32 operands
// The logits of a piece of the vocabulary come from the library's 3xTF32 product and lie in
// the workspace; these passes read them once.

// A block per row: the statistics of logits[row, 0:N] to part[row * nblk + blk]; the
// target's logit if it lies in the piece.
__global__ void __launch_bounds__(256) ce_stats_f32_kernel(const float* __restrict__ logits, int64_t ldl, int64_t N,
                                                           int64_t col0, const int64_t* __restrict__ target,
                                                           float2* part, int nblk, int blk, float* tlogit) {
  __shared__ float2 s_st[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const float* l = logits + row * ldl;
  float m = -INFINITY, s = 0.f;
  for (int64_t c0 = 0; c0 < N; c0 += 2048) {
    float v[8];
    float mx = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = c0 + j * 256 + threadIdx.x;
      v[j] = c < N ? l[c] * kLog2e : -INFINITY;
      mx = fmaxf(mx, v[j]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx;
    s *= ex2(m - ref);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += ex2(v[j] - ref);
    m = mx;
  }
  float2 st = make_float2(m, s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = join_stats(st, make_float2(__shfl_xor_sync(0xffffffffu, st.x, o), __shfl_xor_sync(0xffffffffu, st.y, o)));
  if ((threadIdx.x & 31) == 0) s_st[threadIdx.x >> 5] = st;
  __syncthreads();
  if (threadIdx.x != 0) return;
  st = s_st[0];
  for (int w = 1; w < 8; ++w) st = join_stats(st, s_st[w]);
  part[row * nblk + blk] = st;
  const int64_t y = target[row] - col0;
  if (y >= 0 && y < N) tlogit[row] = l[y] * kLog2e;
}

// logits[row, c] -> grad_row * (softmax - [c is the target]) in place; zeros for tokens
// without a target.
__global__ void __launch_bounds__(256) ce_prob_f32_kernel(float* logits, int64_t ldl, int64_t N, int64_t col0,
                                                          const int64_t* __restrict__ target, int64_t ignore,
                                                          const float2* __restrict__ stats,
                                                          const float* __restrict__ grad,
                                                          const float* __restrict__ count, int reduction) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  float* l = logits + row * ldl;
  const int64_t y = target[row];
  const bool live = y != ignore;
  const float2 st = stats[row];
  float g = 0.f;
  if (live) {
    g = reduction == kReduceNone ? grad[row] : grad[0];
    if (reduction == kReduceMean) g /= count[0];
  }
  const float coef = g / st.y;
  for (int64_t c = threadIdx.x; c < N; c += 256) {
    float x = ex2(fmaf(l[c], kLog2e, -st.x)) * coef;
    if (c + col0 == y) x -= g;
    l[c] = live ? x : 0.f;
  }
}

// x with the rows of tokens without a target zeroed (whatever they hold must not reach the
// gradient of the weight).
__global__ void __launch_bounds__(256) ce_mask_rows_f32_kernel(const float* __restrict__ x, int64_t ldx, float* dst,
                                                               int64_t ldd, int64_t T, int64_t D,
                                                               const int64_t* __restrict__ target, int64_t ignore) {
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const bool live = target[t] != ignore;
    for (int64_t c = threadIdx.x; c < D; c += 256) dst[t * ldd + c] = live ? x[t * ldx + c] : 0.f;
  }
}

// dx += sums (when given), then zeros where a token has no target.
__global__ void __launch_bounds__(256) ce_finish_dx_f32_kernel(float* dx, const float* __restrict__ sums, int64_t T,
                                                               int64_t D, const int64_t* __restrict__ target,
                                                               int64_t ignore, int last) {
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const bool live = !last || target[t] != ignore;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      float v = live ? dx[t * D + c] : 0.f;
      if (live && sums != nullptr) v += sums[t * D + c];
      if (sums != nullptr || !live) dx[t * D + c] = v;
    }
  }
}

}  // namespace tilec
