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
    const float l = mx + logf(s);
    const int t = target[row];
    lse[row] = l;
    // no tile has picked a logit for a label outside the vocabulary: its loss is NaN rather than a wrong number
    losses[row] = t == ignore_index ? 0.0f : (t < 0 || t >= vocab) ? NAN : l - target_logit[row];
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
    const float inv = mean ? 1.0f / static_cast<float>(n) : 1.0f;
    *loss = s * inv;
    *inv_count = inv;
  }
}

inline int launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string(what) + ": " + cudaGetErrorString(e));
  return kOk;
}

}  // namespace

extern "C" int coda_b200_ce_loss(const void* A, int64_t a_stride_m, int64_t a_stride_k, const void* B, int64_t b_stride_k,
                                 int64_t b_stride_n, const int32_t* target, int ignore_index, int mean, float* part_max, float* part_sum,
                                 float* target_logit, float* lse, float* losses, float* loss, float* inv_count, int M, int N, int K,
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
  int rc = launch_gemm<EpiLse<kLseStoreNone>, 0>(a, b, M, N, K, ep, dev_status, st);
  if (rc != kOk) return rc;
  ce_rows_kernel<<<(M + 7) / 8, 256, 0, st>>>(part_max, part_sum, ep.tiles_n, target, target_logit, ignore_index, N, lse, losses, M);
  rc = launch_check("cross-entropy rows launch");
  if (rc != kOk) return rc;
  ce_total_kernel<<<1, 1024, 0, st>>>(losses, target, ignore_index, mean, loss, inv_count, M);
  return launch_check("cross-entropy total launch");
}

extern "C" int coda_b200_gemm_softmax_grad(const void* A, int64_t a_stride_m, int64_t a_stride_k, const void* B, int64_t b_stride_k,
                                           int64_t b_stride_n, const float* lse, const int32_t* target, int ignore_index, int col0, void* G,
                                           int64_t ldg, int M, int N, int K, int* dev_status, void* stream) {
  if (!A || !B || !lse || !target || !G) return fail(kBadArgument, "NULL pointer");
  if (K % 8 != 0) return fail(kBadArgument, "K must be a multiple of 8");
  if (col0 < 0) return fail(kBadArgument, "col0 must not be negative");
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
  return launch_gemm<EpiSoftmaxGrad, 0>(a, b, M, N, K, ep, dev_status, static_cast<cudaStream_t>(stream));
}
