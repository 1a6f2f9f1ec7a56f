// Softmax cross entropy over a vocabulary projection, the passes around its products.
//
//   z = X W^T [T, V],  lse_t = log sum_v exp(z_tv),  loss_t = lse_t - z_t,label(t)
//   d_tv = (g_t + h_t) exp(z_tv - lse_t) - g_t [v = label(t)],  dX = d W,  dW = d^T X
//
// with g, h the gradients of loss and lse.  z is never kept: the forward pass reduces every 128 x 256 tile
// of it in the epilogue of the product (XentStatsFuse in gemm_bf16.cuh) to one (maximum, sum) pair per
// row, and the gradient recomputes it a piece of the vocabulary at a time, turning the accumulators
// into d in the epilogue (XentGradFuse).  d is rounded to bf16 once, because the two products behind it
// take bf16 operands; it is a relative rounding of each value (2^-9), of the size of the rounding of the
// results themselves.
//
// The reference has no loss; the products extend its operator (naive/naive.cpp:6-22).
#pragma once
#include "common.cuh"
#include "tc_common.cuh"
#include "gemm_bf16.cuh"

namespace gemm_b200 {
namespace tc {

constexpr int kXentSlices = 16;   // threads that share one row's column tiles in the finishing pass

// (m, s) with s a sum of exponentials relative to m; an infinite m counts as reference 0 (XentStatsFuse)
__device__ __forceinline__ void xent_merge(float& m, float& s, float pm, float ps) {
  const float now = fmaxf(m, pm);
  const float base = isinf(now) ? 0.f : now;
  s = s * (isinf(m) ? 1.f : expf(m - base)) + ps * (isinf(pm) ? 1.f : expf(pm - base));
  m = now;
}

// Joins the column tiles of every row.  A block owns 32 rows (one per lane, so that the pairs of a column tile are
// read 256 bytes at a time) and cuts the tiles into 16 interleaved slices; always the same order.
// Bound by the read of 8 T ceil(V / 256) bytes, 1/64 of what one bf16 copy of the logits would be.
__global__ void __launch_bounds__(32 * kXentSlices)
xent_finish_kernel(const float2* __restrict__ part, const float* __restrict__ label_logit, const int64_t* __restrict__ labels,
                   float* __restrict__ loss, float* __restrict__ lse, int T, int tiles_n, int V) {
  __shared__ float2 sh[kXentSlices][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_launch_dependents();
  float m = -INFINITY, s = 0.f;
  if (row < T) {
#pragma unroll 4
    for (int t = slice; t < tiles_n; t += kXentSlices) {
      const float2 p = part[(int64_t)t * T + row];
      xent_merge(m, s, p.x, p.y);
    }
  }
  sh[slice][lane] = make_float2(m, s);
  __syncthreads();
  if (slice != 0 || row >= T) return;
  for (int i = 1; i < kXentSlices; ++i) xent_merge(m, s, sh[i][lane].x, sh[i][lane].y);
  const float total = (isinf(m) ? 0.f : m) + logf(s);
  const int64_t label = labels[row];
  lse[row] = total;
  loss[row] = label < 0 ? 0.f : (label >= V ? NAN : total - label_logit[row]);
}

// One block per row: the numbers the gradient epilogue needs, and the row of X for the product d^T X with
// rows of weight zero (padding, whatever it holds) as zeros, since 0 * NaN would reach every row of dW.
__global__ void __launch_bounds__(128)
xent_prepare_kernel(const int64_t* __restrict__ labels, const float* __restrict__ lse, const float* __restrict__ grad_loss,
                    int64_t grad_loss_stride, const float* __restrict__ grad_lse, int64_t grad_lse_stride,
                    const __nv_bfloat16* __restrict__ X, int64_t ldx, XentRow* __restrict__ rows, __nv_bfloat16* __restrict__ Xw, int D,
                    int V) {
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
  uint4* dst = reinterpret_cast<uint4*>(Xw + row * D);
  for (int i = threadIdx.x; i < D / 8; i += 128) dst[i] = live ? src[i] : make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace tc
}  // namespace gemm_b200
