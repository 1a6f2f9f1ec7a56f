// Low-rank adapters of many requests, the passes beside the shared projection.
//
//   y_t = x_t W + s_a (x_t A_a^T) B_a,   a = ids[t]        A [n, R, D], B [n, R, N]
//   dA_a = s_a sum_{t: ids[t] = a} (dy_t B_a^T)^T x_t,     dB_a = s_a sum_{t: ids[t] = a} (x_t A_a^T)^T dy_t
//
// The projection with its second factor is one launch of the GEMM kernel (LoraFuse in gemm_bf16.cuh); here are
// the products with the first factor (V = s x A^T, and dy B^T for the gradient) and the sums over a
// request's tokens.  Both read their long operand once and do little arithmetic on it, so they use
// mma.sync from registers: what bounds them is the read.
//
// The reference has no counterpart; the products extend its operator (naive/naive.cpp:6-22).
#pragma once
#include "common.cuh"
#include "tc_common.cuh"
#include "gemm_bf16.cuh"

namespace gemm_b200 {
namespace tc {

__device__ __forceinline__ void mma_m16n8k16_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                  uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with an accumulator of zero
__device__ __forceinline__ void mma_m16n8k16_bf16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// ---------------------------------------------------------------------------------------
// V[t, r] = s_a sum_k X[t, k] A_a[r, k], a = ids[t], as `terms` bf16 summands of width rp side by side
// (three of them carry 24 bits for FP32 results; one is the ordinary rounding for bf16 results, of the size of
// the rounding of the result).  Rows without an adapter are not written (nothing reads them); a row
// with an id >= n becomes NaN.
//
// Few rows (lora_shrink_kernel): a block has up to four of them and, in a cluster of gridDim.y blocks, a share of K.  Its
// eight warps are dealt out to the rows' adapters first and to K second, so that a block of one request and a block of
// four keep the same number of loads in flight: these sizes are bound by the latency of few, long reads.  A warp
// copies 64 k at a time (cp.async, a 128-byte line by eight lanes) into two stages of its own in shared memory and waits
// for nobody else.  The order of k inside a product is free, so a lane reads sixteen bytes of a row (eight
// consecutive k) as the k pairs of two MMAs, in the same way for X and A.  A row is loaded only under its own
// adapter.  Every warp leaves its rows' sums in its stages; they are added over the warps and then over the cluster,
// in a fixed order.  One row of 4096, rank 16: 6.5 us, most of it the launch and two round trips to memory.
// ---------------------------------------------------------------------------------------
struct ShrinkProblem {
  const __nv_bfloat16* X;
  const __nv_bfloat16* A;
  __nv_bfloat16* V;
  int64_t ldx, lda, stride_a;
  int K;
};
struct ShrinkArgs {
  ShrinkProblem p[2];
  const int32_t* ids;
  const float* scales;   // may be null: 1
  int T, R, n, rp, terms, chunks;   // chunks of 64 ranks
  int rows_per_block;               // lora_shrink_kernel: at most kShrinkFewRows
  // launched behind a kernel whose output is not read here (lora_sort_kernel, which lets it be scheduled only after its own
  // wait): run beside it, and wait for it only at the end, for the kernel behind this one
  bool beside;
};
constexpr int kShrinkWarps = 8, kShrinkK = 64, kShrinkMaxCluster = 8, kShrinkFewRows = 4;

template <int NT8>
struct ShrinkShape {
  static constexpr int ROWS = kShrinkFewRows, COLS = 8 * NT8, LD = COLS + 8;
  static constexpr int STAGE_BYTES = (ROWS + COLS) * 128;                   // rows of 64 k: X, then A
  static constexpr int RING_BYTES = 2 * STAGE_BYTES;                        // per warp
  static constexpr int SMEM_BYTES = kShrinkWarps * RING_BYTES + ROWS * COLS * 4;
  static_assert(ROWS * LD * 4 <= RING_BYTES, "a warp's sums take the place of its stages");
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool in) {
  const int bytes = in ? 16 : 0;   // 0: sixteen zero bytes, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// The last step of both kernels below: the blocks of a cluster add their sums [row][COLS] up in order and write V.
template <int COLS>
__device__ __forceinline__ void shrink_finish(const ShrinkArgs& args, const ShrinkProblem& pr, int chunk, const float* block_sums, const int* id_of,
                                              int row0, int elems) {
  const int rank = blockIdx.y, ranks = gridDim.y;
  if (ranks > 1) {
    cluster_arrive();
    cluster_wait();
  }
  const int64_t ldv = (int64_t)args.terms * args.rp;
  const uint32_t base = smem_u32(block_sums);
  const int share = (elems + ranks - 1) / ranks, e_end = min(elems, (rank + 1) * share);
  for (int e = rank * share + threadIdx.x; e < e_end; e += 32 * kShrinkWarps) {
    const int lr = e / COLS, c = e % COLS, r = chunk * 64 + c;
    const int a = id_of[lr];
    if (a < 0) continue;
    float v = 0.f;
    if (ranks == 1) {
      v = block_sums[e];
    } else {
      float part[kShrinkMaxCluster];
#pragma unroll
      for (int b = 0; b < kShrinkMaxCluster; ++b) part[b] = b < ranks ? ld_shared_cluster_f32(map_to_cta(base + 4u * (uint32_t)e, (uint32_t)b)) : 0.f;
#pragma unroll
      for (int b = 0; b < kShrinkMaxCluster; ++b) v += part[b];
    }
    v = r < args.R ? v : 0.f;
    if (a >= args.n) v = NAN;
    else if (r < args.R && args.scales) v *= args.scales[a];
    __nv_bfloat16* dst = pr.V + (row0 + lr) * ldv + r;
    const long long v_bytes = (long long)args.T * ldv * 2;
    (void)v_bytes;
    for (int t = 0; t < args.terms; ++t) {
      const __nv_bfloat16 h = __float2bfloat16_rn(v);
      if (GEMM_B200_IN_BOUNDS(dst + t * args.rp, pr.V, v_bytes, 2, 50)) dst[t * args.rp] = h;
      const float back = __bfloat162float(h);
      v = isinf(back) ? 0.f : v - back;   // an infinity is whole in its first summand
    }
  }
  if (args.beside) pdl_wait();
  __syncwarp();
  if (ranks > 1) {   // no block leaves while another one reads its sums
    cluster_arrive();
    cluster_wait();
  }
}

// 128-byte rows of a stage; sixteen-byte unit u of row r sits at unit u ^ shrink_swizzle(r): a read takes four units of
// eight rows, and any two neighbouring rows then lie in different halves of the banks.
__device__ __forceinline__ int shrink_swizzle(int row) { return (row & 1) << 2 | (row >> 1 & 3); }

template <int NT8>
__global__ void __launch_bounds__(32 * kShrinkWarps)
lora_shrink_kernel(const __grid_constant__ ShrinkArgs args) {
  using S = ShrinkShape<NT8>;
  extern __shared__ __align__(16) uint8_t shrink_smem[];
  float* block_sums = reinterpret_cast<float*>(shrink_smem + kShrinkWarps * S::RING_BYTES);   // [row][COLS]
  __shared__ int slot_of[S::ROWS], id_of[S::ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = blockIdx.y, ranks = gridDim.y;
  const int chunk = blockIdx.z % args.chunks;
  const ShrinkProblem& pr = args.p[blockIdx.z / args.chunks];
  const int row0 = blockIdx.x * args.rows_per_block;
  const int row_end = min(args.T, row0 + args.rows_per_block);
  if (!args.beside) pdl_wait();
  pdl_launch_dependents();

  TileIds<1> ids;
  ids.load(args.ids, row0, row_end, lane);
  if (warp == 0 && lane < S::ROWS) id_of[lane] = ids.id[0];
  int slots = 0;
  while (ids.next() >= 0) ++slots;
  ids.last = -1;
  const int by_slot = slots > 2 ? 4 : slots > 1 ? 2 : 1, by_k = kShrinkWarps / by_slot;
  // K: a run of steps per block, which the warps of an adapter take in turn
  const int steps = (pr.K + kShrinkK - 1) / kShrinkK, per = (steps + ranks - 1) / ranks;
  const int step0 = min(steps, rank * per) + warp / by_slot, step1 = min(steps, (rank + 1) * per);
  float* warp_sums = reinterpret_cast<float*>(shrink_smem + warp * S::RING_BYTES);            // [row][LD], once the stages are done
  const uint32_t ring = smem_u32(warp_sums);
  const int cr = lane >> 3, cc = lane & 7;   // copies: lane = (row of four, sixteen bytes of eight)

  for (int slot = 0; slot < slots; ++slot) {
    const int a = ids.next();
    if (slot != warp % by_slot) continue;
    float acc[NT8][2];   // rows g < 4 (the products' rows 4 to 7 repeat them, 8 to 15 are nothing)
#pragma unroll
    for (int nt = 0; nt < NT8; ++nt) acc[nt][0] = acc[nt][1] = 0.f;
    if (a < args.n) {
      const bool wanted = __shfl_sync(0xffffffffu, ids.id[0], cr) == a;   // whether this lane's row has the adapter
      const __nv_bfloat16* xp = pr.X + (int64_t)(row0 + cr) * pr.ldx + cc * 8;
      const __nv_bfloat16* ap = pr.A + (int64_t)a * pr.stride_a + (int64_t)(chunk * 64 + cr) * pr.lda + cc * 8;
      const int ranks_left = args.R - chunk * 64 - cr;
      const int64_t a4 = 4 * pr.lda;
      uint32_t dst_of[2];     // where this lane's copies of even and odd groups of four rows go in stage 0
#pragma unroll
      for (int i = 0; i < 2; ++i) dst_of[i] = ring + (uint32_t)(cr * 128 + ((cc ^ shrink_swizzle(i * 4 + cr)) << 4));
      // Rows of another adapter and ranks above R are not copied: what the stage holds there reaches only sums that
      // nobody reads.
      auto load = [&](int step, int stage) {   // one commit group per step, an empty one past the end
        if (step < step1) {
          const int k = step * kShrinkK;
          const bool in = k + cc * 8 < pr.K;   // K ends inside the step: zeros from there on
          const uint32_t to = (uint32_t)(stage * S::STAGE_BYTES);
          if (wanted) cp_async_16(dst_of[0] + to, in ? xp + k : pr.X, in);
          const __nv_bfloat16* src = in ? ap + k : pr.A;
          const int64_t da = in ? a4 : 0;
#pragma unroll
          for (int i = 0; i < S::COLS / 4; ++i, src += da)
            if (i * 4 < ranks_left) cp_async_16(dst_of[i & 1] + to + S::ROWS * 128 + i * 512, src, in);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      load(step0, 0);
      int stage = 0;
      for (int step = step0; step < step1; step += by_k, stage ^= 1) {
        load(step + by_k, stage ^ 1);   // into the stage that every lane is done with: the barrier at the end of the last round
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const uint32_t base = ring + (uint32_t)(stage * S::STAGE_BYTES);
        uint4 x[2], w[2][NT8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          x[half] = ld_shared_16(base + (g & 3) * 128 + (((half * 4 + q) ^ shrink_swizzle(g & 3)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT8; ++nt)
            w[half][nt] = ld_shared_16(base + (S::ROWS + nt * 8 + g) * 128 + (((half * 4 + q) ^ shrink_swizzle(g)) << 4));
        }
        // 64 k at a time in the tensor cores (which cut off low bits of a long running sum), added up in FP32
        float t[NT8][4];
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16_zero(t[nt], x[0].x, 0u, x[0].y, 0u, w[0][nt].x, w[0][nt].y);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[0].z, 0u, x[0].w, 0u, w[0][nt].z, w[0][nt].w);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[1].x, 0u, x[1].y, 0u, w[1][nt].x, w[1][nt].y);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[1].z, 0u, x[1].w, 0u, w[1][nt].z, w[1][nt].w);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) {
          acc[nt][0] += t[nt][0];
          acc[nt][1] += t[nt][1];
        }
        __syncwarp();
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
    const bool mine = __shfl_sync(0xffffffffu, ids.id[0], g) == a;
    if (g < S::ROWS && mine) {
      if (q == 0) slot_of[g] = slot;   // the same value from every warp that writes it
      float* dst = warp_sums + g * S::LD + 2 * q;
#pragma unroll
      for (int nt = 0; nt < NT8; ++nt) *reinterpret_cast<float2*>(dst + nt * 8) = make_float2(acc[nt][0], acc[nt][1]);
    }
  }
  __syncthreads();
  const int elems = (row_end - row0) * S::COLS;
  for (int e = threadIdx.x; e < elems; e += 32 * kShrinkWarps) {
    const int lr = e / S::COLS, c = e % S::COLS;
    if (id_of[lr] < 0) continue;
    float sum = 0.f;
    for (int w = slot_of[lr]; w < kShrinkWarps; w += by_slot)
      sum += reinterpret_cast<const float*>(shrink_smem + w * S::RING_BYTES)[lr * S::LD + c];
    block_sums[e] = sum;
  }
  __syncthreads();
  shrink_finish<S::COLS>(args, pr, chunk, block_sums, id_of, row0, elems);
}

// The same for many rows: 16 * MT of them per block, with TMA.  Every warp takes each eighth step of 64 k and runs two rings of
// its own, X tiles (all rows of the block) and A tiles (one adapter each); one lane asks for another tile once
// the oldest one has been multiplied, so a step costs the warp its reads from shared memory and
// its products.  (With the copies of the kernel above, addresses and predicates were half of the instructions: 8192 x
// 8192, rank 16, one adapter per 512 rows, 41 us; now 33, 4.1 TB/s.)  The adapters of a block share the X tile, each multiplies the
// groups of 16 rows that have it, and a row takes up the products of its own adapter only: by selection, so that
// nothing of another one reaches it.  Bound by the read of X where the rows of a request lie together.
struct ShrinkMaps {
  CUtensorMap x[2], a[2];   // x: box 64 k x ROWS rows; a: [adapters][R][K], box 64 k x COLS ranks
};
template <int MT, int NT8>
struct ShrinkRowsShape {
  static constexpr int ROWS = 16 * MT, COLS = 8 * NT8, LD = COLS + 8;
  static constexpr int A_STAGES = COLS == 16 ? 6 : COLS == 32 ? 3 : 2;      // as many as fit
  static constexpr int X_BYTES = ROWS * 128, A_BYTES = COLS * 128, WARP_BYTES = 2 * X_BYTES + A_STAGES * A_BYTES;
  static constexpr int SUM_BYTES = (kShrinkWarps * ROWS * LD + ROWS * COLS) * 4;   // take the place of the rings
  static constexpr int SMEM_BYTES = 1024 + kShrinkWarps * WARP_BYTES;
  static_assert(SUM_BYTES <= kShrinkWarps * WARP_BYTES && SMEM_BYTES <= 231424, "shared memory budget");
};

template <int MT, int NT8>
__global__ void __launch_bounds__(32 * kShrinkWarps, 1)
lora_shrink_rows_kernel(const __grid_constant__ ShrinkArgs args, const __grid_constant__ ShrinkMaps maps) {
  using S = ShrinkRowsShape<MT, NT8>;
  constexpr int WORDS = (S::ROWS + 31) / 32;
  extern __shared__ uint8_t shrink_rows_raw[];
  uint8_t* smem = shrink_rows_raw + ((1024u - (smem_u32(shrink_rows_raw) & 1023u)) & 1023u);
  __shared__ int id_of[S::ROWS], slot_id[S::ROWS], slot_count;
  __shared__ __align__(8) uint64_t bars[kShrinkWarps * (2 + S::A_STAGES)];
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = blockIdx.y, ranks = gridDim.y;
  const int chunk = blockIdx.z % args.chunks, problem = blockIdx.z / args.chunks;
  const ShrinkProblem& pr = args.p[problem];
  const int row0 = blockIdx.x * S::ROWS, row_end = min(args.T, row0 + S::ROWS);
  const uint32_t x_ring = smem_u32(smem) + warp * S::WARP_BYTES, a_ring = x_ring + 2 * S::X_BYTES;
  const uint32_t x_bar = smem_u32(bars) + warp * 8 * (2 + S::A_STAGES), a_bar = x_bar + 16;
  if (lane == 0) {
    for (int i = 0; i < 2 + S::A_STAGES; ++i) mbar_init(x_bar + 8 * i, 1);
    fence_mbar_init();
  }
  if (!args.beside) pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {   // the block's rows and its distinct adapters, ascending
    TileIds<WORDS> ids;
    ids.load(args.ids, row0, row_end, lane);
#pragma unroll
    for (int w = 0; w < WORDS; ++w)
      if (32 * w + lane < S::ROWS) id_of[32 * w + lane] = ids.id[w];
    int count = 0;
    for (int a = ids.next(); a >= 0 && a < args.n; a = ids.next(), ++count)
      if (lane == 0) slot_id[count] = a;
    if (lane == 0) slot_count = count;
  }
  __syncthreads();
  const int slots = slot_count;
  // Row g of an MMA is row `rho` of its eight rows, for X and A alike: tiles lie in 128-byte swizzled rows (unit u of row r at
  // u ^ (r & 7)), and in this order two neighbouring lanes' rows are read from different halves of the banks.
  const int rho = g >> 1 | (g & 1) << 2;
  int id[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) id[mt][h] = id_of[mt * 16 + h * 8 + rho];
  const int steps = (pr.K + kShrinkK - 1) / kShrinkK, per = (steps + ranks - 1) / ranks;
  const int step0 = min(steps, rank * per) + warp, step1 = min(steps, (rank + 1) * per);
  const bool issuer = elect_one();

  auto load_x = [&](int step, uint32_t buf) {
    if (step < step1 && issuer) {
      mbar_arrive_expect_tx(x_bar + 8 * buf, S::X_BYTES);
      tma_load_3d(x_ring + buf * S::X_BYTES, &maps.x[problem], step * kShrinkK, row0, 0, x_bar + 8 * buf);
    }
  };
  int next_step = step0, next_slot = 0;   // the A tile to ask for next
  auto load_a = [&](uint32_t buf) {
    if (next_step < step1) {
      if (issuer) {
        mbar_arrive_expect_tx(a_bar + 8 * buf, S::A_BYTES);
        tma_load_3d(a_ring + buf * S::A_BYTES, &maps.a[problem], next_step * kShrinkK, chunk * 64, slot_id[next_slot], a_bar + 8 * buf);
      }
      if (++next_slot == slots) { next_slot = 0; next_step += kShrinkWarps; }
    }
  };
  float acc[MT][NT8][4] = {};
  bool failed = false;
  if (slots > 0) {
    load_x(step0, 0);
    load_a(0);
    load_x(step0 + kShrinkWarps, 1);
    for (uint32_t i = 1; i < (uint32_t)S::A_STAGES; ++i) load_a(i);
  }
  const uint32_t unit[2] = {(uint32_t)(q ^ rho) << 4, (uint32_t)((4 + q) ^ rho) << 4};
  uint32_t it = 0, ab = 0, a_phase = 0;
  for (int step = step0; step < step1 && slots > 0 && !failed; step += kShrinkWarps, ++it) {
    const uint32_t xb = it & 1u, xs = x_ring + xb * S::X_BYTES + (uint32_t)rho * 128u;
    if (!mbar_wait_warp(x_bar + 8 * xb, (it >> 1) & 1u, kRoleMma, (int)xb)) { failed = true; break; }
    for (int slot = 0; slot < slots; ++slot) {
      const uint32_t as = a_ring + ab * S::A_BYTES + (uint32_t)rho * 128u;
      if (!mbar_wait_warp(a_bar + 8 * ab, a_phase, kRoleMma, 2 + (int)ab)) { failed = true; break; }
      uint4 w[2][NT8];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) w[half][nt] = ld_shared_16(as + nt * 1024 + unit[half]);
      const int a = slot_id[slot];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (!__any_sync(0xffffffffu, id[mt][0] == a || id[mt][1] == a)) continue;   // none of these 16 rows
        uint4 x[2][2];   // [half of k][rows 0-7, 8-15]
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int h = 0; h < 2; ++h) x[half][h] = ld_shared_16(xs + mt * 2048 + h * 1024 + unit[half]);
        // 64 k at a time in the tensor cores (which cut off low bits of a long running sum), added up in FP32
        float t[NT8][4];
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16_zero(t[nt], x[0][0].x, x[0][1].x, x[0][0].y, x[0][1].y, w[0][nt].x, w[0][nt].y);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[0][0].z, x[0][1].z, x[0][0].w, x[0][1].w, w[0][nt].z, w[0][nt].w);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[1][0].x, x[1][1].x, x[1][0].y, x[1][1].y, w[1][nt].x, w[1][nt].y);
#pragma unroll
        for (int nt = 0; nt < NT8; ++nt) mma_m16n8k16_bf16(t[nt], x[1][0].z, x[1][1].z, x[1][0].w, x[1][1].w, w[1][nt].z, w[1][nt].w);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (id[mt][h] == a) {
#pragma unroll
            for (int nt = 0; nt < NT8; ++nt) {
              acc[mt][nt][2 * h] += t[nt][2 * h];
              acc[mt][nt][2 * h + 1] += t[nt][2 * h + 1];
            }
          }
      }
      // Every fragment read above went into a product that was issued, so it had arrived in its register: the tile
      // may be overwritten.  (Asked for right behind the reads, a tile could land before a read that was still queued.)
      __syncwarp();
      load_a(ab);
      if (++ab == (uint32_t)S::A_STAGES) { ab = 0; a_phase ^= 1u; }
    }
    if (!failed) load_x(step + 2 * kShrinkWarps, xb);   // the same holds for the X tile
  }
  if (failed || aborted()) {   // copies in flight land before shared memory goes away
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
  float* warp_sums = reinterpret_cast<float*>(smem);                                   // [warp][row][LD]
  float* block_sums = warp_sums + kShrinkWarps * S::ROWS * S::LD;                      // [row][COLS]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* dst = warp_sums + (warp * S::ROWS + mt * 16 + h * 8 + rho) * S::LD + q;   // columns 2q, 2q + 1 of the MMA: ranks q, q + 4
#pragma unroll
      for (int nt = 0; nt < NT8; ++nt) {
        dst[nt * 8] = acc[mt][nt][2 * h];
        dst[nt * 8 + 4] = acc[mt][nt][2 * h + 1];
      }
    }
  __syncthreads();
  const int elems = (row_end - row0) * S::COLS;
  for (int e = threadIdx.x; e < elems; e += 32 * kShrinkWarps) {
    const int lr = e / S::COLS, c = e % S::COLS;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kShrinkWarps; ++w) sum += warp_sums[(w * S::ROWS + lr) * S::LD + c];
    block_sums[e] = sum;
  }
  __syncthreads();
  shrink_finish<S::COLS>(args, pr, chunk, block_sums, id_of, row0, elems);
}

// ---------------------------------------------------------------------------------------
// Tokens by adapter, for the gradient: perm[start[a], start[a + 1]) are the rows with id a, ascending.
// One block per adapter scans the ids twice (counts, then places): no atomics, one possible result.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024)
lora_sort_kernel(const int32_t* __restrict__ ids, int T, int n, int32_t* __restrict__ perm, int32_t* __restrict__ start) {
  __shared__ int eq[32], lt[32];
  const int a = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int per = (T + 1023) / 1024 * 32;   // rows per warp, a multiple of 32
  const int r0 = min(T, warp * per), r1 = min(T, r0 + per);
  int n_eq = 0, n_lt = 0;
#pragma unroll 8
  for (int r = r0; r < r1; r += 32) {
    const int id = r + lane < r1 ? ids[r + lane] : -1;
    n_eq += __popc(__ballot_sync(0xffffffffu, id == a));
    n_lt += __popc(__ballot_sync(0xffffffffu, id >= 0 && id < a));
  }
  if (lane == 0) { eq[warp] = n_eq; lt[warp] = n_lt; }
  __syncthreads();
  int at = 0, before = 0, all = 0;
  for (int w = 0; w < 32; ++w) {
    at += lt[w];
    all += eq[w];
    if (w < warp) before += eq[w];
  }
  if (threadIdx.x == 0) {
    start[a] = at;
    if (a == n - 1) start[n] = at + all;
  }
  if (all == 0) return;
  at += before;
  for (int r = r0; r < r1; r += 32) {
    const int id = r + lane < r1 ? ids[r + lane] : -1;
    const unsigned hit = __ballot_sync(0xffffffffu, id == a);
    if (id == a) perm[at + __popc(hit & ((1u << lane) - 1u))] = r + lane;
    at += __popc(hit);
  }
}

// ---------------------------------------------------------------------------------------
// G_a[r, c] = sum over the tokens of a of P[t, r] Q[t, c]: dA from P = s dy B^T and Q = x, dB from P = s x A^T and Q = dy.
//
// The token axis, sorted by adapter, is cut into blocks of equal length whatever the requests' shares are (one
// adapter with every token, or sixty with a few each); a block owns 128 columns and walks the adapters that
// its range touches, 32 tokens per step, the loads running ahead across the adapters' borders.
// A sum that lies inside one block goes straight to the result.  The others, of which a block has two at
// most, leave partial sums: in slot 2 b of block b the one that began in an earlier block, in slot 2 b + 1 the one
// that begins there and goes on; lora_join_kernel adds them in the order of the blocks.  Rows are gathered, so only a request's own tokens
// are ever multiplied: nothing of one request reaches another's gradient.
// ---------------------------------------------------------------------------------------
struct GradProblem {
  const __nv_bfloat16* P;   // [T, terms * rp]
  const __nv_bfloat16* Q;   // [T, cols], pitch ldq
  void* out;                // [n, R, cols]
  float* part;              // [2 * blocks][R][cols]
  int64_t ldq;
  int cols, first_chunk;    // column chunks [first_chunk, ...) of the grid belong to this problem
};
struct GradArgs {
  GradProblem p[2];
  const int32_t* perm;
  const int32_t* start;
  int n, R, blocks;   // blocks: of tokens (gridDim.y of lora_grad_kernel)
};
// Tokens per block, from the number of tokens that have an adapter (known on the device): whole steps of 32 from there on.
__device__ __forceinline__ int grad_block_tokens(int total, int blocks) {
  const int b = (total + blocks - 1) / blocks;
  return b > 32 ? (b + 31) / 32 * 32 : max(4, (b + 3) / 4 * 4);
}
constexpr int kGradCols = 128, kGradTokens = 32, kGradStages = 3, kGradThreads = 128;
constexpr int kGradRows = 8;   // steps whose row indices are held: more than the stages, so that no reader is overtaken

template <int MT, int TERMS>
struct GradShape {
  static constexpr int RP = 16 * MT;
  static constexpr int Q_PITCH = kGradCols * 2 + 16, P_PITCH = RP * TERMS * 2 + 16;   // odd multiples of 16 bytes: ldmatrix without conflicts
  static constexpr int STAGE_BYTES = kGradTokens * (Q_PITCH + P_PITCH);
  static constexpr int SMEM_BYTES = kGradStages * STAGE_BYTES;
  // blocks per SM by shared memory and by registers (80, 128, 168, 255 a thread for 16, 32, 64, 128 ranks)
  static constexpr int BY_SMEM = 231424 / (SMEM_BYTES + 1536), BY_REGS = MT == 1 ? 6 : MT == 2 ? 4 : MT == 4 ? 3 : 2;
  static constexpr int PER_SM = BY_SMEM < BY_REGS ? BY_SMEM : BY_REGS;
};

// Walks the steps of one block: positions [pos, end) of adapter a, at most 32 at a time.
struct GradWalk {
  int a, pos, end, limit;
  __device__ __forceinline__ void settle(const int32_t* start, int n) {   // skip adapters that are used up
    while (a < n && pos >= end) {
      ++a;
      if (a < n) end = min(limit, start[a + 1]);
    }
    if (pos >= limit) a = n;
  }
};

template <int MT, int TERMS, bool OUT_F32>
__global__ void __launch_bounds__(kGradThreads)
lora_grad_kernel(const __grid_constant__ GradArgs args) {
  using S = GradShape<MT, TERMS>;
  extern __shared__ __align__(16) uint8_t grad_smem[];
  __shared__ int row_ring[kGradRows][kGradTokens];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const GradProblem& pr = args.p[(int)blockIdx.x >= args.p[1].first_chunk ? 1 : 0];
  const int c0 = ((int)blockIdx.x - pr.first_chunk) * kGradCols;
  pdl_wait();
  pdl_launch_dependents();
  const int total = args.start[args.n];
  const int block_tokens = grad_block_tokens(total, args.blocks);
  const int lo = blockIdx.y * block_tokens, hi = min(total, lo + block_tokens);
  if (lo >= hi) return;
  // the adapter that position `lo` belongs to: the last one that starts at or before it
  int a0 = 0, a1 = args.n - 1;
  while (a0 < a1) {
    const int mid = (a0 + a1 + 1) >> 1;
    if (args.start[mid] <= lo) a0 = mid; else a1 = mid - 1;
  }
  GradWalk ix{a0, lo, min(hi, args.start[a0 + 1]), hi};   // three walkers: row indices, loads, arithmetic
  ix.settle(args.start, args.n);
  GradWalk cu = ix;

  const uint32_t smem = smem_u32(grad_smem);
  const int64_t ldp = (int64_t)S::RP * TERMS;
  // the rows of the next step of `ix` (lane by lane; -1: none), one step before the loads need them
  auto fetch_rows = [&]() -> int {
    if (ix.a >= args.n) return -1;
    const int cnt = min(kGradTokens, ix.end - ix.pos);
    const int row = lane < cnt ? args.perm[ix.pos + lane] : -1;
    ix.pos += cnt;
    ix.settle(args.start, args.n);
    return row;
  };
  // sixteen threads per token, eight tokens at a time: a thread keeps its columns, so that a copy costs it a row
  // index, one multiplication and the instruction itself
  const int t0 = threadIdx.x / 16, piece = threadIdx.x % 16;
  const bool col_in = c0 + piece * 8 < pr.cols;
  const __nv_bfloat16* q_src = col_in ? pr.Q + c0 + piece * 8 : pr.Q;
  const uint32_t q_dst = (uint32_t)(t0 * S::Q_PITCH + piece * 16), p_dst = (uint32_t)(kGradTokens * S::Q_PITCH + t0 * S::P_PITCH + piece * 16);
  constexpr int PIECES = S::RP * TERMS / 8;   // of a row of P
  auto load_step = [&](int step) {
    const int* rows = row_ring[step % kGradRows];
    const uint32_t base = smem + (step % kGradStages) * S::STAGE_BYTES;
    if (rows[0] >= 0) {   // past the last step: an empty group
#pragma unroll
      for (int i = 0; i < kGradTokens / 8; ++i) {
        const int row = rows[t0 + i * 8];
        const bool in = row >= 0;
        const int64_t at = in ? row : 0;
        cp_async_16(base + q_dst + i * 8 * S::Q_PITCH, q_src + at * pr.ldq, in && col_in);
        const __nv_bfloat16* p_src = pr.P + at * ldp + piece * 8;
#pragma unroll
        for (int j = 0; j < (PIECES + 15) / 16; ++j)
          if (PIECES % 16 == 0 || j < PIECES / 16 || piece + j * 16 < PIECES)
            cp_async_16(base + p_dst + i * 8 * S::P_PITCH + j * 256, p_src + j * 128, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (warp == 0) {
    for (int s = 0; s < kGradStages; ++s) row_ring[s][lane] = fetch_rows();
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kGradStages - 1; ++s) load_step(s);

  float acc[MT][4][4];
  auto clear = [&] {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mt][nt][e] = 0.f;
  };
  clear();
  const int warp_c = warp * 32;
  for (int it = 0; cu.a < args.n; ++it) {
    int next_row = -1;
    if (warp == 0) next_row = fetch_rows();            // step it + kGradStages; used from the next barrier on
    asm volatile("cp.async.wait_group %0;" ::"n"(kGradStages - 2) : "memory");
    __syncthreads();
    load_step(it + kGradStages - 1);                   // into the stage every warp finished with before the barrier
    const uint32_t qs = smem + (it % kGradStages) * S::STAGE_BYTES, ps = qs + kGradTokens * S::Q_PITCH;
    uint32_t b[kGradTokens / 16][2][4];                // 32 tokens x 32 columns
#pragma unroll
    for (int k = 0; k < kGradTokens / 16; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        ldmatrix_x4_trans(b[k][h], qs + (k * 16 + (lane & 15)) * S::Q_PITCH + (warp_c + h * 16 + (lane >> 4) * 8) * 2);
    // a step's products in the tensor cores (which cut off low bits of a long running sum), added up in FP32;
    // two tiles of ranks at a time, so that eight chains of products are under way
    constexpr int G = MT > 1 ? 2 : 1;
#pragma unroll
    for (int m0 = 0; m0 < MT; m0 += G) {
      float tmp[G][4][4];
#pragma unroll
      for (int t = TERMS - 1; t >= 0; --t)
#pragma unroll
        for (int k = 0; k < kGradTokens / 16; ++k)
#pragma unroll
          for (int m = 0; m < G; ++m) {
            uint32_t r[4];    // P^T: 16 ranks x 16 tokens; matrices (tokens 0-7, 8-15) x (ranks 0-7, 8-15)
            ldmatrix_x4_trans(r, ps + (k * 16 + (lane >> 4) * 8 + (lane & 7)) * S::P_PITCH + (t * S::RP + (m0 + m) * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
              if (t == TERMS - 1 && k == 0)
                mma_m16n8k16_bf16_zero(tmp[m][nt], r[0], r[1], r[2], r[3], b[k][nt >> 1][(nt & 1) * 2], b[k][nt >> 1][(nt & 1) * 2 + 1]);
              else
                mma_m16n8k16_bf16(tmp[m][nt], r[0], r[1], r[2], r[3], b[k][nt >> 1][(nt & 1) * 2], b[k][nt >> 1][(nt & 1) * 2 + 1]);
            }
          }
#pragma unroll
      for (int m = 0; m < G; ++m)
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m0 + m][nt][e] += tmp[m][nt][e];
    }
    if (warp == 0) row_ring[(it + kGradStages) % kGradRows][lane] = next_row;
    cu.pos += min(kGradTokens, cu.end - cu.pos);
    if (cu.pos >= cu.end) {   // the adapter's share of this block is complete
      const int a = cu.a;
      const bool whole = args.start[a] >= lo && args.start[a + 1] <= hi;
      const int part_slot = 2 * (int)blockIdx.y + (args.start[a] >= lo ? 1 : 0);
      const long long out_elems = (long long)args.n * args.R * pr.cols;
      (void)out_elems;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = mt * 16 + h * 8 + g;
          if (r >= args.R) continue;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const int c = c0 + warp_c + nt * 8 + 2 * q;
            if (c >= pr.cols) continue;
            const float x = acc[mt][nt][2 * h], y = acc[mt][nt][2 * h + 1];
            if (!whole) {
              float* dst = pr.part + ((int64_t)part_slot * args.R + r) * pr.cols + c;
              if (GEMM_B200_IN_BOUNDS(dst, pr.part, 2ll * args.blocks * args.R * pr.cols * 4, 8, 52)) *reinterpret_cast<float2*>(dst) = make_float2(x, y);
            } else {
              const int64_t at = ((int64_t)a * args.R + r) * pr.cols + c;
              if (!GEMM_B200_IN_BOUNDS(static_cast<char*>(pr.out) + at * (OUT_F32 ? 4 : 2), pr.out, out_elems * (OUT_F32 ? 4 : 2), OUT_F32 ? 8 : 4, 51)) continue;
              if constexpr (OUT_F32) *reinterpret_cast<float2*>(static_cast<float*>(pr.out) + at) = make_float2(x, y);
              else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(pr.out) + at) = __floats2bfloat162_rn(x, y);
            }
          }
        }
      clear();
      cu.settle(args.start, args.n);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Sums the partial sums of adapters whose tokens span blocks, in the order of the blocks, and zeroes the
// gradients of adapters without a token.
template <bool OUT_F32>
__global__ void __launch_bounds__(256)
lora_join_kernel(const __grid_constant__ GradArgs args) {
  const int a = blockIdx.y;
  const GradProblem& pr = args.p[blockIdx.z];
  pdl_wait();
  pdl_launch_dependents();
  const int s0 = args.start[a], s1 = args.start[a + 1];
  const int block_tokens = grad_block_tokens(args.start[args.n], args.blocks);
  const int b0 = s0 / block_tokens, b1 = (s1 - 1) / block_tokens;
  if (s1 > s0 && b0 == b1) return;
  const int64_t elems = (int64_t)args.R * pr.cols;   // a multiple of 8
  for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < elems; e += (int64_t)gridDim.x * 1024) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s1 > s0) {
#pragma unroll 4
      for (int b = b0; b <= b1; ++b) {
        const float4 v = *reinterpret_cast<const float4*>(pr.part + (int64_t)(2 * b + (b == b0 ? 1 : 0)) * elems + e);
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      }
    }
    const int64_t at = (int64_t)a * elems + e;
    if (!GEMM_B200_IN_BOUNDS(static_cast<char*>(pr.out) + at * (OUT_F32 ? 4 : 2), pr.out, (long long)args.n * elems * (OUT_F32 ? 4 : 2), OUT_F32 ? 16 : 8, 53)) continue;
    if constexpr (OUT_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(pr.out) + at) = acc;
    } else {
      __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x, acc.y), hi = __floats2bfloat162_rn(acc.z, acc.w);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(pr.out) + at) =
          make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    }
  }
}

}  // namespace tc
}  // namespace gemm_b200
