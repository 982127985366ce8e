// C-ABI entry points of the cross entropy that walks the vocabulary in pieces and keeps no logits: the loss with its
// per-row log-sum-exp, and the softmax gradient of one piece.  See include/coda_b200.h for the contract.
#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// One warp per row joins the column tiles' (max, sum) and writes the row's log-sum-exp and loss.
__global__ void __launch_bounds__(256) ce_rows_kernel(const float* __restrict__ part_max, const float* __restrict__ part_sum, int tiles_n,
                                                      const int* __restrict__ target, const float* __restrict__ target_logit,
                                                      int ignore_index, int vocab, float* __restrict__ lse, float* __restrict__ losses,
                                                      int M) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= M) return;
  const int t = target[row];
  if (t == ignore_index) {  // such a row may have no partials
    if (lane == 0) lse[row] = losses[row] = 0.0f;
    return;
  }
  const float* pm = part_max + static_cast<long long>(row) * tiles_n;
  const float* ps = part_sum + static_cast<long long>(row) * tiles_n;
  float mx = -INFINITY;
  for (int t = lane; t < tiles_n; t += 32) mx = fmaxf(mx, pm[t]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float s = 0.f;
  for (int t = lane; t < tiles_n; t += 32) s += ps[t] * expf(pm[t] - mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) {
    // No tile has picked a logit for a label outside the vocabulary: its loss is NaN rather than a wrong number, and so is
    // its log-sum-exp, which makes the row's gradient NaN.
    const bool outside = t < 0 || t >= vocab;
    const float l = outside ? NAN : mx + logf(s);
    lse[row] = l;
    losses[row] = outside ? NAN : l - target_logit[row];
  }
}

// One block: the sum of the row losses in a fixed order, the number of rows that count, and with `mean` their quotient
// (NaN when no row counts, as a mean over nothing is).
__global__ void __launch_bounds__(1024) ce_total_kernel(const float* __restrict__ losses, const int* __restrict__ target, int ignore_index,
                                                        int mean, float* __restrict__ loss, float* __restrict__ inv_count, int M) {
  __shared__ float sums[32];
  __shared__ int counts[32];
  float s = 0.f;
  int n = 0;
  for (int i = threadIdx.x; i < M; i += 1024) {
    s += losses[i];
    n += target[i] != ignore_index;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x >> 5] = s;
    counts[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    n = 0;
    for (int i = 0; i < 32; ++i) {
      s += sums[i];
      n += counts[i];
    }
    // the mean over nothing is NaN, and nothing depends on anything
    const float inv = n == 0 ? 0.0f : mean ? 1.0f / static_cast<float>(n) : 1.0f;
    *loss = n == 0 && mean ? NAN : s * inv;
    *inv_count = inv;
  }
}

// What the gradients' products are multiplied by: zero where no row counts, whatever dloss is (1 / 0 behind a sum of nothing).
__global__ void ce_alpha_kernel(const float* __restrict__ dloss, const float* __restrict__ inv_count, float* __restrict__ alpha) {
  *alpha = *inv_count == 0.0f ? 0.0f : *dloss * *inv_count;
}

// ------------------------------------------------------------------ the rows that count
// position[i] = how many rows before i count, or -1 for an ignored one; labels[position[i]] = target[i], the rest of labels
// is ignore_index; *live = how many count.  One block, 1024 rows at a time.
__global__ void __launch_bounds__(1024) ce_positions_kernel(const int* __restrict__ target, int ignore_index, int* __restrict__ position,
                                                            int* __restrict__ labels, int* __restrict__ live, int M) {
  __shared__ int warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int i0 = 0; i0 < M; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    const int t = i < M ? target[i] : ignore_index;
    const bool counts = t != ignore_index;
    const uint32_t ballot = __ballot_sync(0xffffffffu, counts);
    if (lane == 0) warp_sums[warp] = __popc(ballot);
    __syncthreads();
    int sum = lane < warp ? warp_sums[lane] : 0, all = warp_sums[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    const int at = before + sum + __popc(ballot & ((1u << lane) - 1u));
    if (i < M) position[i] = counts ? at : -1;
    if (counts) labels[at] = t;
    before += all;
    __syncthreads();
  }
  for (int i = before + threadIdx.x; i < M; i += 1024) labels[i] = ignore_index;
  if (threadIdx.x == 0) *live = before;
}

// rows[position[i]] = x[i] for the rows that count; the rows behind them up to the next multiple of 64 (which the GEMMs
// work on) are zero.  Block i: row i, and the row that is as far behind the last one.
__global__ void __launch_bounds__(256) ce_gather_kernel(const uint4* __restrict__ x, const int* __restrict__ position,
                                                        const int* __restrict__ live, uint4* __restrict__ rows, int M, int K8) {
  const int i = blockIdx.x, p = position[i], n = *live;
  if (p >= 0)
    for (int c = threadIdx.x; c < K8; c += 256) rows[static_cast<long long>(p) * K8 + c] = __ldcs(x + static_cast<long long>(i) * K8 + c);
  const int end = min(M, (max(n, 1) + 63) / 64 * 64);
  if (n + i < end)
    for (int c = threadIdx.x; c < K8; c += 256) rows[static_cast<long long>(n + i) * K8 + c] = make_uint4(0u, 0u, 0u, 0u);
}

// rows[i] = x[i], zero where row i is ignored: 0 * NaN would take what such a row holds into the weight gradient.
__global__ void __launch_bounds__(256) ce_mask_kernel(const uint4* __restrict__ x, const int* __restrict__ target, int ignore_index,
                                                      uint4* __restrict__ rows, int K8) {
  const int i = blockIdx.x;
  const bool counts = target[i] != ignore_index;
  for (int c = threadIdx.x; c < K8; c += 256)
    rows[static_cast<long long>(i) * K8 + c] = counts ? x[static_cast<long long>(i) * K8 + c] : make_uint4(0u, 0u, 0u, 0u);
}

// dx[i] = rows[position[i]], or zero
__global__ void __launch_bounds__(256) ce_scatter_kernel(const uint4* __restrict__ rows, const int* __restrict__ position,
                                                         uint4* __restrict__ dx, int K8) {
  const int i = blockIdx.x, p = position[i];
  for (int c = threadIdx.x; c < K8; c += 256)
    dx[static_cast<long long>(i) * K8 + c] = p >= 0 ? __ldcs(rows + static_cast<long long>(p) * K8 + c) : make_uint4(0u, 0u, 0u, 0u);
}

inline int launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string(what) + ": " + cudaGetErrorString(e));
  return kOk;
}

}  // namespace

// A whole step, all rows against the rows that count, none / 30 % / 70 % of the rows ignored, in ms: 8192 x 4096 x 128256 26.4
// and 26.9 / 26.3 and 19.2 / 24.8 and 8.6; 2048 x 2048 x 50257 1.40 and 1.39 / 1.34 and 1.11 / 1.29 and 0.76; 1003 x 1032 x
// 32003 0.38 and 0.39 / 0.34 and 0.31 / 0.33 and 0.26.  Smaller products do not repay three more launches (they take one, the
// masked copy of the rows: 512 x 1024 x 32000 0.172 ms, 0.168 without), and with a small vocabulary the copies of the rows weigh too
// much beside them.
extern "C" int coda_b200_ce_compacts(int M, int N, int K) {
  return options().ce_compact.load() != 0 && options().cta_group.load() == 2 && N >= 8192 && 2.0 * M * N * K >= 5e10 ? 1 : 0;
}

extern "C" int coda_b200_ce_compact(const void* x, const int32_t* target, int ignore_index, int32_t* position, int32_t* labels, int32_t* live,
                                    void* rows, int M, int K, void* stream) {
  if (!x || !target || !position || !labels || !live || !rows) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || K <= 0 || K % 8 != 0) return fail(kBadArgument, "M and K must be positive, K a multiple of 8");
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows)) & 15u) != 0) return fail(kBadArgument, "matrices must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ce_positions_kernel<<<1, 1024, 0, st>>>(target, ignore_index, position, labels, live, M);
  const int rc = launch_check("cross-entropy positions launch");
  return rc != kOk ? rc : coda_b200_ce_gather(x, position, live, rows, M, K, stream);
}

extern "C" int coda_b200_ce_gather(const void* x, const int32_t* position, const int32_t* live, void* rows, int M, int K, void* stream) {
  if (!x || !position || !live || !rows) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || K <= 0 || K % 8 != 0) return fail(kBadArgument, "M and K must be positive, K a multiple of 8");
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows)) & 15u) != 0) return fail(kBadArgument, "matrices must be 16-byte aligned");
  ce_gather_kernel<<<M, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint4*>(x), position, live, static_cast<uint4*>(rows), M,
                                                                     K / 8);
  return launch_check("cross-entropy gather launch");
}

extern "C" int coda_b200_ce_mask(const void* x, const int32_t* target, int ignore_index, void* rows, int M, int K, void* stream) {
  if (!x || !target || !rows) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || K <= 0 || K % 8 != 0) return fail(kBadArgument, "M and K must be positive, K a multiple of 8");
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows)) & 15u) != 0) return fail(kBadArgument, "matrices must be 16-byte aligned");
  ce_mask_kernel<<<M, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint4*>(x), target, ignore_index, static_cast<uint4*>(rows),
                                                                   K / 8);
  return launch_check("cross-entropy mask launch");
}

extern "C" int coda_b200_ce_scatter(const void* rows, const int32_t* position, void* dx, int M, int K, void* stream) {
  if (!rows || !position || !dx) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || K <= 0 || K % 8 != 0) return fail(kBadArgument, "M and K must be positive, K a multiple of 8");
  if (((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(rows)) & 15u) != 0) return fail(kBadArgument, "matrices must be 16-byte aligned");
  ce_scatter_kernel<<<M, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint4*>(rows), position, static_cast<uint4*>(dx), K / 8);
  return launch_check("cross-entropy scatter launch");
}

namespace {
// a launch whose rows, or contraction, end at *live
template <class Epi, int kLive, bool kAMn, bool kBMn>
int launch_live(const void* a, long long lda, const void* b, long long ldb, int M, int N, int K, typename Epi::Params& ep, const int* live,
                int* dev_status, cudaStream_t stream) {
  LaunchOptions opt = launch_options();
  opt.ragged = true;  // a piece of the vocabulary may have any number of columns
  if (opt.cta_group != 2) return fail(kBadArgument, "products of counted rows are built for CTA pairs only (cta_group = 2)");
  if (M <= 0 || N <= 0 || K <= 0) return fail(kBadArgument, "GEMM extents must be positive");
  if (dev_status == nullptr) return fail(kBadArgument, "device status word is required");
  ep.use_tma = opt.epi_tma;
  typename ProLive<kLive>::Params pp;
  pp.live = live;
  return launch_gemm_cfg<2, 256, kAMn, kBMn, Epi, ProLive<kLive>>(a, lda, b, ldb, M, N, K, ep, dev_status, stream, opt, pp);
}

template <typename OutT>
int run_live(const void* A, int64_t lda, const void* B, int64_t ldb, const float* C, void* D, int64_t ldd, const float* alpha, const int* live,
             int along_depth, int M, int N, int K, int* dev_status, cudaStream_t stream) {
  using Epi = EpiStore<OutT, Act::kNone>;
  typename Epi::Params ep;
  ep.D = static_cast<OutT*>(D);
  ep.ldd = ldd;
  ep.alpha = alpha;
  ep.C = C;
  ep.ldc = ldd;
  ep.c_is_fp32 = 1;
  const int rc = make_tmap_out(&ep.tm_d, ep.D, N, M, ldd);
  if (rc != kOk) return rc;
  if (along_depth) return launch_live<Epi, 2, true, true>(A, lda, B, ldb, M, N, K, ep, live, dev_status, stream);
  return launch_live<Epi, 1, false, true>(A, lda, B, ldb, M, N, K, ep, live, dev_status, stream);
}
}  // namespace

extern "C" int coda_b200_gemm_live(const void* A, int64_t lda, const void* B, int64_t ldb, const float* C, void* D, int64_t ldd, int d_is_fp32,
                                   const float* alpha, const int32_t* live, int along_depth, int M, int N, int K, int* dev_status,
                                   void* stream) {
  if (!A || !B || !D || !live) return fail(kBadArgument, "NULL pointer");
  if (N % 8 != 0 || ldd % 8 != 0 || ldd < N) return fail(kBadArgument, "N and ldd must be multiples of 8 with ldd >= N");
  if ((reinterpret_cast<uintptr_t>(D) & 15u) != 0 || (reinterpret_cast<uintptr_t>(C) & 15u) != 0)
    return fail(kBadArgument, "C and D must be 16-byte aligned");
  if (lda < (along_depth ? M : K) || ldb < N) return fail(kBadArgument, "a leading dimension is smaller than its row");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d_is_fp32) return run_live<float>(A, lda, B, ldb, C, D, ldd, alpha, live, along_depth, M, N, K, dev_status, st);
  return run_live<__nv_bfloat16>(A, lda, B, ldb, C, D, ldd, alpha, live, along_depth, M, N, K, dev_status, st);
}

extern "C" int coda_b200_ce_loss(const void* A, int64_t a_stride_m, int64_t a_stride_k, const void* B, int64_t b_stride_k,
                                 int64_t b_stride_n, const int32_t* target, int ignore_index, int mean, const int32_t* live,
                                 float* part_max, float* part_sum, float* target_logit, float* lse, float* losses, float* loss, float* inv_count, int M, int N, int K,
                                 int* dev_status, void* stream) {
  if (!A || !B || !target || !part_max || !part_sum || !target_logit || !lse || !losses || !loss || !inv_count)
    return fail(kBadArgument, "NULL pointer");
  if (K % 8 != 0) return fail(kBadArgument, "K must be a multiple of 8");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  EpiLse<kLseStoreNone>::Params ep;
  memset(&ep.tm_p, 0, sizeof(ep.tm_p));
  ep.P = nullptr;
  ep.ldp = 0;
  ep.part_max = part_max;
  ep.part_sum = part_sum;
  ep.tiles_n = coda_b200_lse_tiles(N);
  ep.target = target;
  ep.target_logit = target_logit;
  ep.row_scale = nullptr;
  ep.part_sz = nullptr;
  Operand a{A, a_stride_m, a_stride_k};
  Operand b{B, b_stride_n, b_stride_k};
  int rc;
  if (live == nullptr) rc = launch_gemm<EpiLse<kLseStoreNone>, 0>(a, b, M, N, K, ep, dev_status, st);
  else if (a_stride_k != 1 || b_stride_k != 1) rc = fail(kBadLayout, "counted rows need both operands contiguous along the contraction");
  else rc = launch_live<EpiLse<kLseStoreNone>, 1, false, false>(A, a_stride_m, B, b_stride_n, M, N, K, ep, live, dev_status, st);
  if (rc != kOk) return rc;
  ce_rows_kernel<<<(M + 7) / 8, 256, 0, st>>>(part_max, part_sum, ep.tiles_n, target, target_logit, ignore_index, N, lse, losses, M);
  rc = launch_check("cross-entropy rows launch");
  if (rc != kOk) return rc;
  ce_total_kernel<<<1, 1024, 0, st>>>(losses, target, ignore_index, mean, loss, inv_count, M);
  return launch_check("cross-entropy total launch");
}

extern "C" int coda_b200_ce_alpha(const float* dloss, const float* inv_count, float* alpha, void* stream) {
  if (!dloss || !inv_count || !alpha) return fail(kBadArgument, "NULL pointer");
  ce_alpha_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(dloss, inv_count, alpha);
  return launch_check("cross-entropy factor launch");
}

extern "C" int coda_b200_gemm_softmax_grad(const void* A, int64_t a_stride_m, int64_t a_stride_k, const void* B, int64_t b_stride_k,
                                           int64_t b_stride_n, const float* lse, const int32_t* target, int ignore_index, int col0,
                                           const int32_t* live, void* G, int64_t ldg, int M, int N, int K, int* dev_status, void* stream) {
  if (!A || !B || !lse || !target || !G) return fail(kBadArgument, "NULL pointer");
  if (K % 8 != 0) return fail(kBadArgument, "K must be a multiple of 8");
  if (col0 < 0) return fail(kBadArgument, "col0 must not be negative");
  if (live != nullptr && (a_stride_k != 1 || b_stride_k != 1))
    return fail(kBadLayout, "counted rows need both operands contiguous along the contraction");
  if ((reinterpret_cast<uintptr_t>(G) & 15u) != 0 || ldg % 8 != 0 || ldg < N)
    return fail(kBadArgument, "G must be 16-byte aligned with ldg a multiple of 8 and >= N");
  EpiSoftmaxGrad::Params ep;
  ep.G = static_cast<__nv_bfloat16*>(G);
  ep.ldg = ldg;
  ep.lse = lse;
  ep.target = target;
  ep.ignore_index = ignore_index;
  ep.col0 = col0;
  const int rc = make_tmap_out(&ep.tm_g, ep.G, N, M, ldg);
  if (rc != kOk) return rc;
  Operand a{A, a_stride_m, a_stride_k};
  Operand b{B, b_stride_n, b_stride_k};
  if (live == nullptr) return launch_gemm<EpiSoftmaxGrad, 0>(a, b, M, N, K, ep, dev_status, static_cast<cudaStream_t>(stream));
  return launch_live<EpiSoftmaxGrad, 1, false, false>(A, a_stride_m, B, b_stride_n, M, N, K, ep, live, dev_status,
                                                      static_cast<cudaStream_t>(stream));
}
