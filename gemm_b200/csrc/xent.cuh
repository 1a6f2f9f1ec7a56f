// Softmax cross entropy over a vocabulary projection, the passes around its products.
//
//   z = X W^T [T, V],  lse_t = log sum_v exp(z_tv),  loss_t = lse_t - z_t,label(t)
//   d_tv = (g_t + h_t) exp(z_tv - lse_t) - g_t [v = label(t)],  dX = d W,  dW = d^T X
//
// with g, h the gradients of loss and lse.  z is never kept: the forward pass reduces it in the epilogue of the
// product (XentStatsFuse in gemm_bf16.cuh) to one (maximum, sum) pair per row and 128 columns, and the gradient recomputes it a piece of the vocabulary at a time, turning the accumulators
// into d in the epilogue (XentGradFuse).  d is rounded to bf16, because the two products behind it take bf16
// operands: a relative rounding of each value (2^-9 at most), of the size of the rounding of the results
// themselves and independent from value to value.  With few rows one of these roundings, that of the label's
// entry, is most of a row's error, so up to 64 rows are kept as two bf16 summands (16 bits), one below
// the other: rows T + t of d for dX = d W, whose two halves are added in FP32, and tokens T + t for dW = d^T X.  W is
// still read once and dW written once, which is what bounds these sizes.
//
// The reference has no loss; the products extend its operator (naive/naive.cpp:6-22).
#pragma once
#include "common.cuh"
#include "tc_common.cuh"
#include "gemm_bf16.cuh"

namespace gemm_b200 {
namespace tc {

// (m, s) with s a sum of exponentials relative to m; an infinite m counts as reference 0 (XentStatsFuse)
__device__ __forceinline__ float xent_weight(float m, float base) { return isinf(m) ? 1.f : expf(m - base); }
__device__ __forceinline__ void xent_merge(float& m, float& s, float pm, float ps) {
  const float now = fmaxf(m, pm);
  const float base = isinf(now) ? 0.f : now;
  s = s * xent_weight(m, base) + ps * xent_weight(pm, base);
  m = now;
}

// Joins the column groups of every row, always in the same order.  A block of 1024 threads owns ROWS rows: thread
// (slice, row) takes every 1024 / ROWS-th group, eight loads at a time.  With many rows 32 of them read 256 bytes of a group
// together; with few, the threads go along the vocabulary instead (one row of 131072 columns as one slice
// of 16 took 14 us, as 1024 slices 5 us).  Bound by the read of 8 T ceil(V / 128) bytes, 1/32 of
// a bf16 copy of the logits.
constexpr int kXentFinishThreads = 1024;
template <int ROWS>
__global__ void __launch_bounds__(kXentFinishThreads)
xent_finish_kernel(const float2* __restrict__ part, const float* __restrict__ label_logit, const int64_t* __restrict__ labels,
                   float* __restrict__ loss, float* __restrict__ lse, int T, int groups, int V) {
  constexpr int SLICES = kXentFinishThreads / ROWS, WARPS = kXentFinishThreads / 32;
  __shared__ float2 sh[ROWS][WARPS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int in_block = threadIdx.x % ROWS, slice = threadIdx.x / ROWS;
  const int row = blockIdx.x * ROWS + in_block;
  pdl_wait();
  pdl_launch_dependents();
  float m = -INFINITY, s = 0.f;
  if (row < T) {
    for (int t0 = slice; t0 < groups; t0 += 8 * SLICES) {
      float2 p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = t0 + j * SLICES;
        p[j] = t < groups ? part[(int64_t)t * T + row] : make_float2(-INFINITY, 0.f);
      }
      float now = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) now = fmaxf(now, p[j].x);
      const float base = isinf(now) ? 0.f : now;
      s *= xent_weight(m, base);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += p[j].y * xent_weight(p[j].x, base);
      m = now;
    }
  }
#pragma unroll
  for (int o = ROWS; o < 32; o *= 2) {
    const float pm = __shfl_xor_sync(0xffffffffu, m, o), ps = __shfl_xor_sync(0xffffffffu, s, o);
    xent_merge(m, s, pm, ps);
  }
  if (lane < ROWS) sh[in_block][warp] = make_float2(m, s);
  __syncthreads();
  if (warp >= ROWS) return;
  m = sh[warp][lane].x;                 // warp w: row w of the block
  s = sh[warp][lane].y;
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    const float pm = __shfl_xor_sync(0xffffffffu, m, o), ps = __shfl_xor_sync(0xffffffffu, s, o);
    xent_merge(m, s, pm, ps);
  }
  const int out = blockIdx.x * ROWS + warp;
  if (lane != 0 || out >= T) return;
  const float total = (isinf(m) ? 0.f : m) + logf(s);
  if (!GEMM_B200_IN_BOUNDS(lse + out, lse, (long long)T * 4, 4, 42)) return;
  const int64_t label = labels[out];
  lse[out] = total;
  loss[out] = label < 0 ? 0.f : (label >= V ? NAN : total - label_logit[out]);
}

// One block per row: the numbers the gradient epilogue needs, and the row of X for the product d^T X with
// rows of weight zero (padding, whatever it holds) as zeros, since 0 * NaN would reach every row of dW.
__global__ void __launch_bounds__(128)
xent_prepare_kernel(const int64_t* __restrict__ labels, const float* __restrict__ lse, const float* __restrict__ grad_loss,
                    int64_t grad_loss_stride, const float* __restrict__ grad_lse, int64_t grad_lse_stride,
                    const __nv_bfloat16* __restrict__ X, int64_t ldx, XentRow* __restrict__ rows, __nv_bfloat16* __restrict__ Xw, int copies,
                    int D, int V) {
  const int64_t row = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t label = labels[row];
  float g = label < 0 ? 0.f : grad_loss[row * grad_loss_stride];
  if (label >= V) g = NAN;
  const float a = g + (grad_lse ? grad_lse[row * grad_lse_stride] : 0.f);
  const bool live = a != 0.f || g != 0.f;
  if (threadIdx.x == 0) {
    XentRow r;
    r.neg_lse_log2e = -lse[row] * 1.4426950408889634f;
    r.a = a;
    r.b = g;
    r.label = label >= 0 && label < V ? (int)label : -1;
    rows[row] = r;
  }
  const uint4* src = reinterpret_cast<const uint4*>(X + row * ldx);
  for (int c = 0; c < copies; ++c) {   // one below the other: [copies][T][D]
    uint4* dst = reinterpret_cast<uint4*>(Xw + (row + (int64_t)c * gridDim.x) * D);
    for (int i = threadIdx.x; i < D / 8; i += 128) dst[i] = live ? src[i] : make_uint4(0u, 0u, 0u, 0u);
  }
}

}  // namespace tc
}  // namespace gemm_b200
