// Host side of the operators fused to a BF16 projection: softmax cross entropy over a vocabulary
// (xent.cuh) and low-rank adapters of many requests (lora.cuh).  Part of tc_gemm.cu, which holds the launch
// helpers and the one status word of the tensor-core kernels.
//
// Scratch is the caller's in every entry point: nothing is kept between calls, so calls on different
// streams, and graphs captured from them, share nothing.
#pragma once

namespace gemm_b200 {
namespace tc {

// Launches a plain kernel as a programmatic dependent launch (each waits before it touches global memory).
template <class Kern, class... Args>
static int launch_plain(Kern kern, dim3 grid, int threads, int smem_bytes, int cluster_y, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  static const bool pdl = env_int("GEMM_B200_PDL", 1) != 0;
  int n = 0;
  if (cluster_y > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = 1;
    attrs[n].val.clusterDim.y = (unsigned)cluster_y;
    attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = (unsigned)n;
  GEMM_B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  launch_counter().fetch_add(1, std::memory_order_relaxed);
  return GEMM_B200_OK;
}

// Opts a kernel in to more shared memory than the default 48 KB (of which it may use some statically), once per device.
template <class Kern>
static int allow_smem(Kern kern, int smem_bytes, const DeviceInfo& di) {
  if (smem_bytes <= 40 * 1024) return GEMM_B200_OK;
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> done;
  std::lock_guard<std::mutex> lk(mu);
  int& have = done[std::pair<int, const void*>(di.dev, reinterpret_cast<const void*>(kern))];
  if (have < smem_bytes) {
    GEMM_B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes));
    have = smem_bytes;
  }
  return GEMM_B200_OK;
}

// Cuts a caller's scratch buffer into 256-byte aligned pieces; with a null base it only counts.
struct Carver {
  char* base;
  size_t used = 0;
  template <class T>
  T* take(int64_t count) {
    used = (used + 255) & ~(size_t)255;
    T* p = reinterpret_cast<T*>(base + used);
    used += (size_t)(count > 0 ? count : 0) * sizeof(T);
    return base ? p : nullptr;
  }
};

static int check_scratch(const char* who, const void* scratch, size_t have, size_t need) {
  if (need > 0 && (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0))
    return fail(GEMM_B200_ERR_INVALID_ARG, "%s: scratch must be a 256-byte aligned device buffer", who);
  if (have < need) return fail(GEMM_B200_ERR_INVALID_ARG, "%s: scratch holds %zu bytes, %zu needed", who, have, need);
  return GEMM_B200_OK;
}
static int check_blackwell(const char* who, DeviceInfo* di) {
  if (int rc = device_info(di)) return rc;
  if (di->cc_major != 10)
    return fail(GEMM_B200_ERR_UNSUPPORTED, "%s: device has compute capability %d.x, need 10.x (sm_100a)", who, di->cc_major);
  return GEMM_B200_OK;
}
static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// More than one round of long units: hand them out at run time (the rule of pick_bf16_config).
static bool bf16_pairs_dynamic(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t units = ceil_div64(M, 2 * kBlockM) * ceil_div64(N, kBlockN);
  return units > sms / 2 && K >= 6144;
}

// A product of one row tile, 128 x 256 tiles of single CTAs, the box of A by the number of rows.
template <int A_ROWS>
using Bf16_row_tile = Bf16Cfg<1, A_ROWS == 32 ? 5 : 4, 1, false, 1, 2, kBlockN, false, 0, A_ROWS>;
template <bool B_MN, bool OUT_F32, class Fuse>
static int launch_row_tile(const Bf16Args& a, const Fuse& fuse) {
  if (a.M <= 32) return launch_bf16_fused<Bf16_row_tile<32>, B_MN, OUT_F32, false, Fuse>(a, fuse);
  if (a.M <= 64) return launch_bf16_fused<Bf16_row_tile<64>, B_MN, OUT_F32, false, Fuse>(a, fuse);
  return launch_bf16_fused<Bf16_1cta_tma, B_MN, OUT_F32, false, Fuse>(a, fuse);
}

// =========================================================================================
// Softmax cross entropy
// =========================================================================================
// One row tile streams W once, with a box of X that fits the rows (A_ROWS in gemm_bf16.cuh).
template <int A_ROWS>
using Xent_1cta = Bf16Cfg<1, A_ROWS == 128 ? 4 : 5, 0, false, 1, 0, kBlockN, false, 8, A_ROWS>;
using Xent_2cta = Bf16Cfg<2, 7, 0, true, 1, 0, kBlockN, false, 8>;
using Xent_2cta_dyn = Bf16Cfg<2, 7, 0, true, 1, 0, kBlockN, true, 8>;

struct XentScratch {
  float2* part;
  float* label_logit;
  size_t bytes;
  XentScratch(void* base, int64_t T, int64_t V) {
    Carver c{static_cast<char*>(base)};
    part = c.take<float2>(ceil_div64(V, kXentCols) * T);
    label_logit = c.take<float>(T);
    bytes = c.used;
  }
};

static int xent_sizes(const char* who, int64_t T, int64_t V, int64_t D, int64_t ldx, int64_t ldw) {
  if (T < 0 || V < 1 || D < 1) return fail(GEMM_B200_ERR_INVALID_ARG, "%s: T must not be negative, V and D must be positive", who);
  if (ldx < D || ldw < D)
    return fail(GEMM_B200_ERR_INVALID_ARG, "%s: leading dimension smaller than the row (ldx=%lld ldw=%lld)", who, (long long)ldx, (long long)ldw);
  // columns of the last tile and of the epilogue's look-ahead stay within 31 bits
  if (T > 0x7fffffff || V > 0x7ffffc00 || D > 0x7fffffff) return fail(GEMM_B200_ERR_TOO_LARGE, "%s: a dimension exceeds 2^31-1", who);
  return GEMM_B200_OK;
}

// The gradient works on pieces of the vocabulary whose d (bf16) takes at most this much scratch, but of 4096 columns at
// least: every piece but the first adds T x D FP32 values to dX, which a shorter product would not hide.
constexpr int64_t kXentPieceBytes = 256ll << 20, kXentMinPiece = 4096;

struct XentGradPlan {
  int halves;                 // bf16 summands of d, one below the other: two for up to 64 rows, one row tile (xent.cuh)
  int64_t pieces, piece;      // columns of the vocabulary per piece (the last may be shorter)
  int dx_splits, dw_splits;   // K ranges of the products dX = d W (K: the piece) and dW = d^T X (K: the tokens)
  bool dx_acc;                // dX is summed in FP32 slices: more than one piece, K ranges, or two halves
  XentGradPlan(int64_t T, int64_t V, int64_t D, int sms) {
    halves = 2 * T <= kBlockM ? 2 : 1;
    const int64_t rows = halves * T;
    int64_t most = kXentPieceBytes / (2 * (rows > 0 ? rows : 1)) / kBlockN * kBlockN;
    if (most < kXentMinPiece) most = kXentMinPiece;
    pieces = ceil_div64(V, most);
    piece = pieces == 1 ? V : ceil_div64(ceil_div64(V, pieces), kBlockN) * kBlockN;
    pieces = ceil_div64(V, piece);
    dx_splits = bf16_auto_splits(rows, D, piece, sms);
    dw_splits = bf16_auto_splits(piece, D, rows, sms);
    dx_acc = pieces > 1 || dx_splits > 1 || halves > 1;
  }
};
struct XentGradScratch {
  XentRow* rows;
  __nv_bfloat16 *xw, *d;
  int64_t ldd;
  float *dx, *dw;
  size_t bytes;
  XentGradScratch(void* base, int64_t T, int64_t D, const XentGradPlan& p) {
    Carver c{static_cast<char*>(base)};
    ldd = ceil_div64(p.piece, 8) * 8;
    rows = c.take<XentRow>(T);
    xw = c.take<__nv_bfloat16>(p.halves * T * D);
    d = c.take<__nv_bfloat16>(p.halves * T * ldd);
    dx = c.take<float>(p.dx_acc ? (int64_t)p.dx_splits * p.halves * T * D : 0);
    dw = c.take<float>(p.dw_splits > 1 ? (int64_t)p.dw_splits * p.piece * D : 0);
    bytes = c.used;
  }
};

// FP32 tiles of A @ B into the slices at a.C: stored (first) or added to what is there.
template <class Fuse>
static int launch_bf16_slices(const Bf16Args& a, const Fuse& fuse, int sms) {
  if (a.M <= kBlockM) return launch_row_tile<true, true>(a, fuse);
  if (a.k_splits == 1 && bf16_pairs_dynamic(a.M, a.N, a.K, sms))
    return launch_bf16_fused<Bf16_2cta_tma_m_dyn, true, true, false, Fuse>(a, fuse);
  return launch_bf16_fused<Bf16_2cta_tma_m, true, true, false, Fuse>(a, fuse);
}

static int xent_entry(const void* X, const void* W, const int64_t* labels, float* loss, float* lse, int64_t T, int64_t V, int64_t D,
                      int64_t ldx, int64_t ldw, void* scratch, size_t scratch_bytes, void* stream) {
  if (int rc = xent_sizes("gemm_bf16_xent", T, V, D, ldx, ldw)) return rc;
  if (T == 0) return GEMM_B200_OK;
  if (!X || !W || !labels || !loss || !lse) return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_xent: null pointer");
  if (!aligned16(X) || !aligned16(W) || ldx % 8 != 0 || ldw % 8 != 0)
    return fail(GEMM_B200_ERR_ALIGNMENT, "gemm_bf16_xent: X and W must be 16-byte aligned, ldx and ldw multiples of 8 (ldx=%lld ldw=%lld)",
                (long long)ldx, (long long)ldw);
  const XentScratch ws(scratch, T, V);
  if (int rc = check_scratch("gemm_bf16_xent", scratch, scratch_bytes, ws.bytes)) return rc;
  DeviceInfo di;
  if (int rc = check_blackwell("gemm_bf16_xent", &di)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Bf16Args a{X, W, nullptr, T, V, D, ldx, ldw, V, st};
  const XentStatsFuse fuse{ws.part, ws.label_logit, labels};
  int rc;
  if (T <= 32) rc = launch_bf16_fused<Xent_1cta<32>, false, true>(a, fuse);
  else if (T <= 64) rc = launch_bf16_fused<Xent_1cta<64>, false, true>(a, fuse);
  else if (T <= kBlockM) rc = launch_bf16_fused<Xent_1cta<128>, false, true>(a, fuse);
  else if (bf16_pairs_dynamic(T, V, D, di.sms)) rc = launch_bf16_fused<Xent_2cta_dyn, false, true>(a, fuse);
  else rc = launch_bf16_fused<Xent_2cta, false, true>(a, fuse);
  if (rc) return rc;
  const int groups = (int)ceil_div64(V, kXentCols);
  auto finish = [&](auto kern, int rows) {
    return launch_plain(kern, dim3((unsigned)ceil_div64(T, rows)), kXentFinishThreads, 0, 1, st, (const float2*)ws.part,
                        (const float*)ws.label_logit, labels, loss, lse, (int)T, groups, (int)V);
  };
  return T >= 2048 ? finish(xent_finish_kernel<32>, 32) : T >= 64 ? finish(xent_finish_kernel<4>, 4) : finish(xent_finish_kernel<1>, 1);
}

static int xent_grad_entry(const void* X, const void* W, const int64_t* labels, const float* lse, const float* grad_loss,
                           int64_t grad_loss_stride, const float* grad_lse, int64_t grad_lse_stride, void* dX, void* dW, int64_t T,
                           int64_t V, int64_t D, int64_t ldx, int64_t ldw, int64_t lddx, int64_t lddw, void* scratch,
                           size_t scratch_bytes, void* stream) {
  if (int rc = xent_sizes("gemm_bf16_xent_grad", T, V, D, ldx, ldw)) return rc;
  if (lddx < D || lddw < D)
    return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_xent_grad: leading dimension smaller than the row (lddx=%lld lddw=%lld)",
                (long long)lddx, (long long)lddw);
  if (grad_loss_stride < 0 || grad_lse_stride < 0) return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_xent_grad: negative stride");
  if (!dW || (T > 0 && (!X || !W || !labels || !lse || !grad_loss || !dX)))
    return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_xent_grad: null pointer");
  if (!aligned16(X) || !aligned16(W) || !aligned16(dX) || !aligned16(dW) || D % 8 != 0 || ldx % 8 != 0 || ldw % 8 != 0 ||
      lddx % 8 != 0 || lddw % 8 != 0)
    return fail(GEMM_B200_ERR_ALIGNMENT,
                "gemm_bf16_xent_grad: X, W, dX and dW must be 16-byte aligned, D and the leading dimensions multiples of 8 "
                "(D=%lld ldx=%lld ldw=%lld lddx=%lld lddw=%lld)",
                (long long)D, (long long)ldx, (long long)ldw, (long long)lddx, (long long)lddw);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    GEMM_B200_CUDA_TRY(cudaMemset2DAsync(dW, (size_t)lddw * 2, 0, (size_t)D * 2, (size_t)V, st));
    return GEMM_B200_OK;
  }
  DeviceInfo di;
  if (int rc = check_blackwell("gemm_bf16_xent_grad", &di)) return rc;
  const XentGradPlan plan(T, V, D, di.sms);
  const XentGradScratch ws(scratch, T, D, plan);
  if (int rc = check_scratch("gemm_bf16_xent_grad", scratch, scratch_bytes, ws.bytes)) return rc;
  if (log_enabled())
    fprintf(stderr, "[gemm_b200] gemm_bf16_xent_grad T=%lld V=%lld D=%lld -> %lld pieces of %lld, K ranges %d (dX) %d (dW)\n", (long long)T,
            (long long)V, (long long)D, (long long)plan.pieces, (long long)plan.piece, plan.dx_splits, plan.dw_splits);
  if (int rc = launch_plain(xent_prepare_kernel, dim3((unsigned)T), 128, 0, 1, st, labels, lse, grad_loss, grad_loss_stride, grad_lse,
                            grad_lse_stride, static_cast<const __nv_bfloat16*>(X), ldx, ws.rows, ws.xw, plan.halves, (int)D, (int)V))
    return rc;
  int dx_slices = 1;
  for (int64_t v0 = 0; v0 < V; v0 += plan.piece) {
    const int64_t n = V - v0 < plan.piece ? V - v0 : plan.piece;
    const char* Wp = static_cast<const char*>(W) + v0 * ldw * 2;
    // d of the piece
    const Bf16Args z{X, Wp, ws.d, T, n, D, ldx, ldw, ws.ldd, st};
    XentGradFuse fuse = {};
    fuse.rows = ws.rows;
    fuse.col0 = (int)v0;
    fuse.low = plan.halves > 1;
    int rc;
    if (fuse.low && (rc = make_map_3d(&fuse.tmLow, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ws.d + T * ws.ldd, T, n, ws.ldd, 1, T * ws.ldd, 64, 32,
                                      CU_TENSOR_MAP_SWIZZLE_128B)))   // the box of the epilogue's stores
      return rc;
    if (T <= kBlockM) rc = launch_row_tile<false, false>(z, fuse);
    else if (bf16_pairs_dynamic(T, n, D, di.sms)) rc = launch_bf16_fused<Bf16_2cta_tma_m_dyn, false, false>(z, fuse);
    else rc = launch_bf16_fused<Bf16_2cta_tma_m, false, false>(z, fuse);
    if (rc) return rc;
    // dX (+)= d W
    const int64_t rows = plan.halves * T;
    Bf16Args gx{ws.d, Wp, dX, rows, D, n, ws.ldd, ldw, lddx, st};
    if (!plan.dx_acc && T <= kBlockM) {
      rc = launch_row_tile<true, false>(gx, NoFuse());
    } else if (!plan.dx_acc) {
      rc = kBf16Configs[pick_bf16_config(T, D, n, di.sms)].launch[GEMM_B200_B_ROW_MAJOR_KN][GEMM_B200_OUT_BF16](gx);
    } else {
      gx.C = ws.dx;
      gx.ldc = D;
      gx.k_splits = plan.dx_splits;
      if (v0 == 0) {
        const int64_t num_kb = ceil_div64(n, kBlockK);
        dx_slices = (int)ceil_div64(num_kb, ceil_div64(num_kb, plan.dx_splits));
        rc = launch_bf16_slices(gx, NoFuse(), di.sms);
      } else {
        rc = launch_bf16_slices(gx, AddFuse(), di.sms);   // a later, shorter piece may leave the last slices as they are
      }
    }
    if (rc) return rc;
    // dW of the piece's rows = d^T X
    Bf16Args gw{ws.d, ws.xw, static_cast<char*>(dW) + v0 * lddw * 2, n, D, rows, ws.ldd, D, lddw, st};
    if (plan.dw_splits > 1) {
      rc = launch_bf16_splitk(gw, GEMM_B200_B_ROW_MAJOR_KN, GEMM_B200_OUT_BF16, plan.dw_splits, ws.dw, /*a_mn=*/true);
    } else {
      // A K of a few blocks: the store of dW bounds the product, and single CTAs (two per pair to drain
      // accumulators) store faster (dW [32001, 2048] of 67 tokens 36 us against 45, [131072, 4096] of 16 190
      // against 286); from 512 tokens on pairs are as fast ([50001, 1024] of 509 tokens 51 / 49).
      const int config = rows <= 256 ? (int)kBf16Cfg1cta : pick_bf16_config(n, D, rows, di.sms);
      rc = GEMM_B200_ERR_UNSUPPORTED;
      for (const Bf16AtEntry& e : kBf16AtConfigs)
        if (e.config == config) rc = e.launch[GEMM_B200_B_ROW_MAJOR_KN][GEMM_B200_OUT_BF16](gw);
    }
    if (rc) return rc;
  }
  // slice i of half h starts at row (2 i + h) T of the scratch: twice as many slices of T rows
  if (plan.dx_acc) return launch_splitk_reduce(ws.dx, T, D, plan.halves * dx_slices, dX, lddx, GEMM_B200_OUT_BF16, st);
  return GEMM_B200_OK;
}

// =========================================================================================
// Low-rank adapters
// =========================================================================================
constexpr int64_t kLoraMaxRank = 128;

static int lora_rp(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }
// bf16 summands per value of V: FP32 results keep 24 bits of it, bf16 results the 8 they are rounded to themselves.  With
// few rows and a low rank these roundings do not average out (one row, rank 1: one of them is the whole
// error of the adapter's term), and there the summands cost nothing: three fit into the K block of one.
static int lora_terms(int64_t T, int64_t R, int out_dtype) { return out_dtype == GEMM_B200_OUT_F32 || (T <= 64 && R <= 16) ? 3 : 1; }
// the gradient's: with few tokens its time is that of its launches
static int lora_grad_terms(int64_t T, int out_dtype) { return out_dtype == GEMM_B200_OUT_F32 || T <= 64 ? 3 : 1; }

static int lora_sizes(const char* who, int64_t T, int64_t N, int64_t D, int64_t R, int64_t n, int64_t ldx, int64_t lda, int64_t stride_a,
                      int64_t ldb, int64_t stride_b, int out_dtype) {
  if (T < 0 || N < 1 || D < 1 || R < 1 || n < 1)
    return fail(GEMM_B200_ERR_INVALID_ARG, "%s: T must not be negative, N, D, R and the number of adapters must be positive", who);
  if (out_dtype != GEMM_B200_OUT_BF16 && out_dtype != GEMM_B200_OUT_F32) return fail(GEMM_B200_ERR_INVALID_ARG, "%s: out_dtype %d", who, out_dtype);
  if (R > kLoraMaxRank) return fail(GEMM_B200_ERR_TOO_LARGE, "%s: rank %lld above %lld", who, (long long)R, (long long)kLoraMaxRank);
  if (T > 0x7fffffff || N > 0x7fffffff || D > 0x7fffffff || n > 0x7fffffff)
    return fail(GEMM_B200_ERR_TOO_LARGE, "%s: a dimension exceeds 2^31-1", who);
  if (ldx < D || lda < D || ldb < N || stride_a < (R - 1) * lda + D || stride_b < (R - 1) * ldb + N)
    return fail(GEMM_B200_ERR_INVALID_ARG, "%s: a leading dimension or stride is smaller than its matrix", who);
  if (D % 8 != 0 || N % 8 != 0 || ldx % 8 != 0 || lda % 8 != 0 || ldb % 8 != 0 || stride_a % 8 != 0 || stride_b % 8 != 0)
    return fail(GEMM_B200_ERR_ALIGNMENT, "%s: D, N, the leading dimensions and the strides must be multiples of 8", who);
  return GEMM_B200_OK;
}

// K over the blocks of a cluster: the largest that keeps the grid within `places`, as long as every block keeps a step
// of its eight warps.
static int shrink_cluster(int64_t blocks, int64_t max_k, int64_t places) {
  int ks = 1;
  while (ks < kShrinkMaxCluster && blocks * 2 * ks <= places && max_k / (kShrinkK * kShrinkWarps) >= 2 * ks) ks *= 2;
  return ks;
}

template <int NT8>
static int launch_shrink_few(ShrinkArgs args, int problems, int64_t max_k, const DeviceInfo& di, cudaStream_t st) {
  using S = ShrinkShape<NT8>;
  auto kern = lora_shrink_kernel<NT8>;
  if (int rc = allow_smem(kern, S::SMEM_BYTES, di)) return rc;
  // a block per row, so that every adapter streams on its own; from 65 rows on four share a block (97 rows of 32
  // requests, rank 113: 32 us with sixteen, whose adapters a warp takes one after another)
  args.rows_per_block = args.T <= 64 ? 1 : kShrinkFewRows;
  const int64_t blocks = ceil_div64(args.T, args.rows_per_block), z = problems * args.chunks;
  const int ks = shrink_cluster(blocks * z, max_k, 4 * (int64_t)di.sms);   // rows without an adapter leave at once
  return launch_plain(kern, dim3((unsigned)blocks, (unsigned)ks, (unsigned)z), 32 * kShrinkWarps, S::SMEM_BYTES, ks, st, args);
}

template <int MT, int NT8>
static int launch_shrink_rows(ShrinkArgs args, int problems, int64_t max_k, const DeviceInfo& di, cudaStream_t st) {
  using S = ShrinkRowsShape<MT, NT8>;
  auto kern = lora_shrink_rows_kernel<MT, NT8>;
  if (int rc = allow_smem(kern, S::SMEM_BYTES, di)) return rc;
  args.rows_per_block = S::ROWS;
  ShrinkMaps maps;
  for (int i = 0; i < 2; ++i) {
    const ShrinkProblem& p = args.p[i < problems ? i : 0];
    if (int rc = make_map_3d(&maps.x[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.X, args.T, p.K, p.ldx, 1, args.T * p.ldx, kShrinkK, S::ROWS,
                             CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
    if (int rc = make_map_3d(&maps.a[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.A, args.R, p.K, p.lda, args.n, p.stride_a, kShrinkK, S::COLS,
                             CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
  }
  const int64_t blocks = ceil_div64(args.T, S::ROWS), z = problems * args.chunks;
  const int ks = shrink_cluster(blocks * z, max_k, di.sms);                // a block has its SM to itself
  return launch_plain(kern, dim3((unsigned)blocks, (unsigned)ks, (unsigned)z), 32 * kShrinkWarps, S::SMEM_BYTES, ks, st, args, maps);
}

static int lora_shrink(ShrinkArgs args, int problems, int64_t max_k, const DeviceInfo& di, cudaStream_t st) {
  args.chunks = args.rp > 64 ? 2 : 1;
  const int cols = args.rp > 64 ? 64 : args.rp;
  if (args.T < 512)
    return cols == 16   ? launch_shrink_few<2>(args, problems, max_k, di, st)
           : cols == 32 ? launch_shrink_few<4>(args, problems, max_k, di, st)
                        : launch_shrink_few<8>(args, problems, max_k, di, st);
  return cols == 16   ? launch_shrink_rows<4, 2>(args, problems, max_k, di, st)
         : cols == 32 ? launch_shrink_rows<4, 4>(args, problems, max_k, di, st)
                      : launch_shrink_rows<2, 8>(args, problems, max_k, di, st);
}

struct LoraScratch {
  __nv_bfloat16* V;
  float* slices;
  size_t bytes;
  LoraScratch(void* base, int64_t T, int64_t N, int64_t R, int terms, int splits) {
    Carver c{static_cast<char*>(base)};
    V = c.take<__nv_bfloat16>(T * terms * lora_rp(R));
    slices = c.take<float>(splits > 1 ? (int64_t)splits * T * N : 0);
    bytes = c.used;
  }
};

// the tile shapes of FP32 results: accumulators drained every 512 of K
template <int A_ROWS>
using Lora_row_tile_f32 = Bf16Cfg<1, A_ROWS == 32 ? 5 : 4, 1, false, 1, 1, kBlockN, false, 8, A_ROWS>;
using Lora_2cta_f32 = Bf16Cfg<2, 6, 1, true, 1, 1, kBlockN, false, 8>;
using Lora_2cta_f32_dyn = Bf16Cfg<2, 6, 1, true, 1, 1, kBlockN, true, 8>;

// f32: an FP32 result; otherwise bf16, or the FP32 slices of one that is split over K
template <bool B_MN>
static int launch_lora(const Bf16Args& a, const LoraFuse& fuse, bool f32, int sms) {
  if (a.M <= kBlockM) {
    if (!f32) return a.k_splits > 1 ? launch_row_tile<B_MN, true>(a, fuse) : launch_row_tile<B_MN, false>(a, fuse);
    if (a.M <= 32) return launch_bf16_fused<Lora_row_tile_f32<32>, B_MN, true>(a, fuse);
    if (a.M <= 64) return launch_bf16_fused<Lora_row_tile_f32<64>, B_MN, true>(a, fuse);
    return launch_bf16_fused<Lora_row_tile_f32<128>, B_MN, true>(a, fuse);
  }
  if (a.k_splits > 1) return f32 ? launch_bf16_fused<Lora_2cta_f32, B_MN, true>(a, fuse) : launch_bf16_fused<Bf16_2cta_tma_m, B_MN, true>(a, fuse);
  if (bf16_pairs_dynamic(a.M, a.N, a.K, sms))
    return f32 ? launch_bf16_fused<Lora_2cta_f32_dyn, B_MN, true>(a, fuse) : launch_bf16_fused<Bf16_2cta_tma_m_dyn, B_MN, false>(a, fuse);
  return f32 ? launch_bf16_fused<Lora_2cta_f32, B_MN, true>(a, fuse) : launch_bf16_fused<Bf16_2cta_tma_m, B_MN, false>(a, fuse);
}

// K ranges of the projection: the estimate of bf16_auto_splits with the adapters' K blocks, which the ranges share, beside
// those of D.  How many adapters a row tile has is known on the device only: a decoding batch (one row tile) is taken
// to have one per row, longer ones (prompts, whose rows of one request lie together) half of that.
static int lora_splits(int64_t T, int64_t N, int64_t D, int64_t R, int64_t n, int terms, int sms) {
  const bool pair = bf16_splitk_pairs(T);
  const int64_t rows = pair ? 2 * kBlockM : kBlockM, rp = lora_rp(R);
  const int64_t tiles = ceil_div64(T, rows) * ceil_div64(N, kBlockN), slots = pair ? sms / 2 : sms;
  const int64_t num_kb = ceil_div64(D, kBlockK);
  int64_t ads = T < rows ? T : rows;
  if (n < ads) ads = n;
  if (pair) ads = (ads + 1) / 2;
  const int64_t ad_kb = rp <= 64 ? ceil_div64(ads, 64 / rp) * ceil_div64(terms * rp, 64) : ads * terms * (rp / 64);
  if (3 * tiles >= 2 * slots || num_kb + ad_kb < 32) return 1;
  const double t_kb = pair ? 0.30 : 0.39, slice_us = (double)T * (double)N * 8.0 / 7.8e6;
  double best_cost = (double)(num_kb + ad_kb) * t_kb;   // less than one round: see above
  int best = 1;
  for (int s = 2; s <= 32; ++s) {
    const int64_t kb_per = ceil_div64(num_kb, s), per = kb_per + ceil_div64(ad_kb, s);
    if (kb_per < 2 || per < 8) break;                                    // at least 512 of K per range
    if ((double)s * (double)T * (double)N * 4.0 > 268435456.0) break;   // scratch of at most 256 MiB
    if (ceil_div64(num_kb, kb_per) != s) continue;                      // no empty range
    const double cost = (double)ceil_div64(tiles * s, slots) * (double)per * t_kb + s * slice_us + 6.0;
    if (cost < best_cost) { best_cost = cost; best = s; }
  }
  return best;
}

static int lora_entry(const void* X, const void* W, const void* A, const void* B, const int32_t* ids, const float* scales, void* Y,
                      int64_t T, int64_t N, int64_t D, int64_t R, int64_t n, int64_t ldx, int64_t ldw, int64_t lda, int64_t stride_a,
                      int64_t ldb, int64_t stride_b, int64_t ldy, int w_layout, int out_dtype, void* scratch, size_t scratch_bytes,
                      void* stream) {
  if (int rc = lora_sizes("gemm_bf16_lora", T, N, D, R, n, ldx, lda, stride_a, ldb, stride_b, out_dtype)) return rc;
  if (w_layout != GEMM_B200_B_ROW_MAJOR_KN && w_layout != GEMM_B200_B_ROW_MAJOR_NK)
    return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_lora: w_layout %d", w_layout);
  if (ldw < (w_layout == GEMM_B200_B_ROW_MAJOR_KN ? N : D) || ldy < N)
    return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_lora: leading dimension smaller than the row (ldw=%lld ldy=%lld)", (long long)ldw, (long long)ldy);
  if (T == 0) return GEMM_B200_OK;
  if (!X || !W || !A || !B || !ids || !Y) return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_lora: null pointer");
  const int c_elem = out_dtype == GEMM_B200_OUT_F32 ? 4 : 2;
  if (!aligned16(X) || !aligned16(W) || !aligned16(A) || !aligned16(B) || !aligned16(Y) || ldw % 8 != 0 || (ldy * c_elem) % 16 != 0)
    return fail(GEMM_B200_ERR_ALIGNMENT, "gemm_bf16_lora: X, W, A, B and Y must be 16-byte aligned, ldw a multiple of 8, ldy*sizeof(Y) of 16 bytes");
  DeviceInfo di;
  if (int rc = check_blackwell("gemm_bf16_lora", &di)) return rc;
  const int terms = lora_terms(T, R, out_dtype), rp = lora_rp(R), splits = lora_splits(T, N, D, R, n, terms, di.sms);
  const LoraScratch ws(scratch, T, N, R, terms, splits);
  if (int rc = check_scratch("gemm_bf16_lora", scratch, scratch_bytes, ws.bytes)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  ShrinkArgs sa = {};
  sa.p[0] = ShrinkProblem{static_cast<const __nv_bfloat16*>(X), static_cast<const __nv_bfloat16*>(A), ws.V, ldx, lda, stride_a, (int)D};
  sa.p[1] = sa.p[0];
  sa.ids = ids;
  sa.scales = scales;
  sa.T = (int)T;
  sa.R = (int)R;
  sa.n = (int)n;
  sa.rp = rp;
  sa.terms = terms;
  if (int rc = lora_shrink(sa, 1, D, di, st)) return rc;

  LoraFuse fuse;
  if (int rc = make_map_3d(&fuse.tmV, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ws.V, T, (int64_t)terms * rp, (int64_t)terms * rp, 1,
                           T * terms * rp, kBlockK, T <= 32 ? 32 : T <= 64 ? 64 : kBlockM, CU_TENSOR_MAP_SWIZZLE_128B))   // the box of X's tiles
    return rc;
  if (int rc = make_map_3d(&fuse.tmAd, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, B, R, N, ldb, n, stride_b, 64, rp < 64 ? rp : 64,
                           CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  fuse.ids = ids;
  fuse.rp = rp;
  fuse.terms = terms;
  Bf16Args a{X, W, Y, T, N, D, ldx, ldw, ldy, st};
  const bool f32 = out_dtype == GEMM_B200_OUT_F32;
  if (splits > 1) {
    a.C = ws.slices;
    a.ldc = N;
    a.k_splits = splits;
  }
  const int rc = w_layout == GEMM_B200_B_ROW_MAJOR_KN ? launch_lora<true>(a, fuse, f32, di.sms) : launch_lora<false>(a, fuse, f32, di.sms);
  if (rc || splits == 1) return rc;
  return launch_splitk_reduce(ws.slices, T, N, splits, Y, ldy, out_dtype, st);
}

static int lora_grad_per_sm(int rp, int terms) {
  if (terms == 1)
    return rp == 16 ? GradShape<1, 1>::PER_SM : rp == 32 ? GradShape<2, 1>::PER_SM : rp == 64 ? GradShape<4, 1>::PER_SM : GradShape<8, 1>::PER_SM;
  return rp == 16 ? GradShape<1, 3>::PER_SM : rp == 32 ? GradShape<2, 3>::PER_SM : rp == 64 ? GradShape<4, 3>::PER_SM : GradShape<8, 3>::PER_SM;
}

struct LoraGradPlan {
  int64_t chunks_d, chunks_n, blocks;
  LoraGradPlan(int64_t T, int64_t N, int64_t D, int64_t R, int terms, int sms) {
    chunks_d = ceil_div64(D, kGradCols);
    chunks_n = ceil_div64(N, kGradCols);
    // Blocks of tokens so that the grid fills one, two or three rounds of the resident thread blocks best (672 thread
    // blocks on 444 places: a third of the second round idle), but not below four tokens.
    const int64_t chunks = chunks_d + chunks_n, slots = (int64_t)sms * lora_grad_per_sm(lora_rp(R), terms), most = ceil_div64(T > 0 ? T : 1, 4);
    blocks = 1;
    double best = 0;
    for (int rounds = 1; rounds <= 3; ++rounds) {
      int64_t b = rounds * slots / chunks;
      if (b < 1) b = 1;
      if (b > most) b = most;
      const double fill = (double)(b * chunks) / (double)(ceil_div64(b * chunks, slots) * slots);
      if (fill > best + 0.03) { best = fill; blocks = b; }
    }
  }
};
struct LoraGradScratch {
  __nv_bfloat16 *u, *v;
  int32_t *perm, *start;
  float *part_a, *part_b;
  size_t bytes;
  LoraGradScratch(void* base, int64_t T, int64_t N, int64_t D, int64_t R, int64_t n, int terms, const LoraGradPlan& p) {
    Carver c{static_cast<char*>(base)};
    u = c.take<__nv_bfloat16>(T * terms * lora_rp(R));
    v = c.take<__nv_bfloat16>(T * terms * lora_rp(R));
    perm = c.take<int32_t>(T);
    start = c.take<int32_t>(n + 1);
    const int64_t parts = p.blocks > 1 ? 2 * p.blocks : 0;   // each block's first and last sum may be partial
    part_a = c.take<float>(parts * R * D);
    part_b = c.take<float>(parts * R * N);
    bytes = c.used;
  }
};

template <int MT, int TERMS, bool F32>
static int launch_lora_grad(const GradArgs& ga, const LoraGradPlan& plan, const DeviceInfo& di, cudaStream_t st) {
  auto kern = lora_grad_kernel<MT, TERMS, F32>;
  constexpr int smem = GradShape<MT, TERMS>::SMEM_BYTES;
  if (int rc = allow_smem(kern, smem, di)) return rc;
  if (int rc = launch_plain(kern, dim3((unsigned)(plan.chunks_d + plan.chunks_n), (unsigned)plan.blocks), kGradThreads, smem, 1, st, ga))
    return rc;
  // about eight blocks per SM over the adapters and both operands
  const int64_t most = ceil_div64((int64_t)ga.R * (ga.p[0].cols > ga.p[1].cols ? ga.p[0].cols : ga.p[1].cols), 1024);
  int64_t bx = ceil_div64(8 * (int64_t)di.sms, 2 * (int64_t)ga.n);
  if (bx > most) bx = most;
  return launch_plain(lora_join_kernel<F32>, dim3((unsigned)bx, (unsigned)ga.n, 2), 256, 0, 1, st, ga);
}

template <int TERMS, bool F32>
static int launch_lora_grad_rp(int rp, const GradArgs& ga, const LoraGradPlan& plan, const DeviceInfo& di, cudaStream_t st) {
  return rp == 16   ? launch_lora_grad<1, TERMS, F32>(ga, plan, di, st)
         : rp == 32 ? launch_lora_grad<2, TERMS, F32>(ga, plan, di, st)
         : rp == 64 ? launch_lora_grad<4, TERMS, F32>(ga, plan, di, st)
                    : launch_lora_grad<8, TERMS, F32>(ga, plan, di, st);
}

static int lora_grad_entry(const void* X, const void* dY, const void* A, const void* B, const int32_t* ids, const float* scales, void* dA,
                           void* dB, int64_t T, int64_t N, int64_t D, int64_t R, int64_t n, int64_t ldx, int64_t lddy, int64_t lda,
                           int64_t stride_a, int64_t ldb, int64_t stride_b, int out_dtype, void* scratch, size_t scratch_bytes,
                           void* stream) {
  if (int rc = lora_sizes("gemm_bf16_lora_grad", T, N, D, R, n, ldx, lda, stride_a, ldb, stride_b, out_dtype)) return rc;
  if (n > 65535) return fail(GEMM_B200_ERR_TOO_LARGE, "gemm_bf16_lora_grad: more than 65535 adapters");
  if (lddy < N) return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_lora_grad: leading dimension smaller than the row (lddy=%lld)", (long long)lddy);
  if (!dA || !dB || (T > 0 && (!X || !dY || !A || !B || !ids))) return fail(GEMM_B200_ERR_INVALID_ARG, "gemm_bf16_lora_grad: null pointer");
  if (!aligned16(X) || !aligned16(dY) || !aligned16(A) || !aligned16(B) || !aligned16(dA) || !aligned16(dB) || lddy % 8 != 0)
    return fail(GEMM_B200_ERR_ALIGNMENT, "gemm_bf16_lora_grad: X, dY, A, B, dA and dB must be 16-byte aligned, lddy a multiple of 8");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t c_elem = out_dtype == GEMM_B200_OUT_F32 ? 4 : 2;
  if (T == 0) {
    GEMM_B200_CUDA_TRY(cudaMemsetAsync(dA, 0, (size_t)n * R * D * c_elem, st));
    GEMM_B200_CUDA_TRY(cudaMemsetAsync(dB, 0, (size_t)n * R * N * c_elem, st));
    return GEMM_B200_OK;
  }
  DeviceInfo di;
  if (int rc = check_blackwell("gemm_bf16_lora_grad", &di)) return rc;
  const int terms = lora_grad_terms(T, out_dtype), rp = lora_rp(R);
  const LoraGradPlan plan(T, N, D, R, terms, di.sms);
  const LoraGradScratch ws(scratch, T, N, D, R, n, terms, plan);
  if (int rc = check_scratch("gemm_bf16_lora_grad", scratch, scratch_bytes, ws.bytes)) return rc;

  if (int rc = launch_plain(lora_sort_kernel, dim3((unsigned)n), 1024, 0, 1, st, ids, (int)T, (int)n, ws.perm, ws.start)) return rc;
  ShrinkArgs sa = {};
  sa.p[0] = ShrinkProblem{static_cast<const __nv_bfloat16*>(dY), static_cast<const __nv_bfloat16*>(B), ws.u, lddy, ldb, stride_b, (int)N};
  sa.p[1] = ShrinkProblem{static_cast<const __nv_bfloat16*>(X), static_cast<const __nv_bfloat16*>(A), ws.v, ldx, lda, stride_a, (int)D};
  sa.ids = ids;
  sa.scales = scales;
  sa.T = (int)T;
  sa.R = (int)R;
  sa.n = (int)n;
  sa.rp = rp;
  sa.terms = terms;
  sa.beside = true;
  if (int rc = lora_shrink(sa, 2, D > N ? D : N, di, st)) return rc;

  GradArgs ga = {};
  ga.p[0] = GradProblem{ws.u, static_cast<const __nv_bfloat16*>(X), dA, ws.part_a, ldx, (int)D, 0};
  ga.p[1] = GradProblem{ws.v, static_cast<const __nv_bfloat16*>(dY), dB, ws.part_b, lddy, (int)N, (int)plan.chunks_d};
  ga.perm = ws.perm;
  ga.start = ws.start;
  ga.n = (int)n;
  ga.R = (int)R;
  ga.blocks = (int)plan.blocks;
  if (out_dtype == GEMM_B200_OUT_F32) return launch_lora_grad_rp<3, true>(rp, ga, plan, di, st);
  return terms > 1 ? launch_lora_grad_rp<3, false>(rp, ga, plan, di, st) : launch_lora_grad_rp<1, false>(rp, ga, plan, di, st);
}

static int current_sms() {
  DeviceInfo di;
  return device_info(&di) ? 0 : di.sms;
}

}  // namespace tc
}  // namespace gemm_b200

extern "C" size_t gemm_b200_gemm_bf16_xent_scratch_bytes(int64_t T, int64_t V) {
  if (T <= 0 || V <= 0) return 0;
  return gemm_b200::tc::XentScratch(nullptr, T, V).bytes;
}
extern "C" int gemm_b200_gemm_bf16_xent(const void* X, const void* W, const int64_t* labels, float* loss, float* lse, int64_t T, int64_t V,
                                        int64_t D, int64_t ldx, int64_t ldw, void* scratch, size_t scratch_bytes, void* stream) {
  return gemm_b200::tc::xent_entry(X, W, labels, loss, lse, T, V, D, ldx, ldw, scratch, scratch_bytes, stream);
}
extern "C" size_t gemm_b200_gemm_bf16_xent_grad_scratch_bytes(int64_t T, int64_t V, int64_t D) {
  using namespace gemm_b200::tc;
  const int sms = current_sms();
  if (T <= 0 || V <= 0 || D <= 0 || sms <= 0) return 0;
  return XentGradScratch(nullptr, T, D, XentGradPlan(T, V, D, sms)).bytes;
}
extern "C" int gemm_b200_gemm_bf16_xent_grad(const void* X, const void* W, const int64_t* labels, const float* lse, const float* grad_loss,
                                             int64_t grad_loss_stride, const float* grad_lse, int64_t grad_lse_stride, void* dX, void* dW,
                                             int64_t T, int64_t V, int64_t D, int64_t ldx, int64_t ldw, int64_t lddx, int64_t lddw,
                                             void* scratch, size_t scratch_bytes, void* stream) {
  return gemm_b200::tc::xent_grad_entry(X, W, labels, lse, grad_loss, grad_loss_stride, grad_lse, grad_lse_stride, dX, dW, T, V, D, ldx, ldw,
                                        lddx, lddw, scratch, scratch_bytes, stream);
}
extern "C" size_t gemm_b200_gemm_bf16_lora_scratch_bytes(int64_t T, int64_t N, int64_t D, int64_t R, int64_t adapters, int out_dtype) {
  using namespace gemm_b200::tc;
  const int sms = current_sms();
  if (T <= 0 || N <= 0 || D <= 0 || R <= 0 || R > kLoraMaxRank || adapters <= 0 || sms <= 0) return 0;
  const int terms = lora_terms(T, R, out_dtype);
  return LoraScratch(nullptr, T, N, R, terms, lora_splits(T, N, D, R, adapters, terms, sms)).bytes;
}
extern "C" int gemm_b200_gemm_bf16_lora(const void* X, const void* W, const void* A, const void* B, const int32_t* ids, const float* scales,
                                        void* Y, int64_t T, int64_t N, int64_t D, int64_t R, int64_t adapters, int64_t ldx, int64_t ldw,
                                        int64_t lda, int64_t stride_a, int64_t ldb, int64_t stride_b, int64_t ldy, int w_layout,
                                        int out_dtype, void* scratch, size_t scratch_bytes, void* stream) {
  return gemm_b200::tc::lora_entry(X, W, A, B, ids, scales, Y, T, N, D, R, adapters, ldx, ldw, lda, stride_a, ldb, stride_b, ldy, w_layout,
                                   out_dtype, scratch, scratch_bytes, stream);
}
extern "C" size_t gemm_b200_gemm_bf16_lora_grad_scratch_bytes(int64_t T, int64_t N, int64_t D, int64_t R, int64_t adapters, int out_dtype) {
  using namespace gemm_b200::tc;
  const int sms = current_sms();
  if (T <= 0 || N <= 0 || D <= 0 || R <= 0 || R > kLoraMaxRank || adapters <= 0 || sms <= 0) return 0;
  const int terms = lora_grad_terms(T, out_dtype);
  return LoraGradScratch(nullptr, T, N, D, R, adapters, terms, LoraGradPlan(T, N, D, R, terms, sms)).bytes;
}
extern "C" int gemm_b200_gemm_bf16_lora_grad(const void* X, const void* dY, const void* A, const void* B, const int32_t* ids,
                                             const float* scales, void* dA, void* dB, int64_t T, int64_t N, int64_t D, int64_t R,
                                             int64_t adapters, int64_t ldx, int64_t lddy, int64_t lda, int64_t stride_a, int64_t ldb,
                                             int64_t stride_b, int out_dtype, void* scratch, size_t scratch_bytes, void* stream) {
  return gemm_b200::tc::lora_grad_entry(X, dY, A, B, ids, scales, dA, dB, T, N, D, R, adapters, ldx, lddy, lda, stride_a, ldb, stride_b,
                                        out_dtype, scratch, scratch_bytes, stream);
}
