// C-ABI entry point of the projection of e4m3 rows by an e4m3 weight.  See include/coda_b200.h for the contract.
#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// ------------------------------------------------------------------ few rows
// The product for a handful of rows of x is a stream of the weight through the SMs, bound by HBM: a tile of the GEMM core
// would keep 16 to 48 CTA pairs busy and fill most of its A operand with zeros.  Here a block owns 16 weight rows and its
// 8 warps share out the contraction in steps of 64, several steps in flight; the warps' sums are added in shared memory
// in a fixed order.
//
// The product itself is mma.sync m16n8k32 with the weight rows as M and the rows of x as N (kTiles tiles of 8).  A thread
// holds, for weight rows g and g + 8 (g = lane / 4), 16 consecutive bytes at 16 (lane % 4) of the step, and the same 16
// bytes of row g of x.  The instruction wants bytes 4 t .. 4 t + 3 and 16 + 4 t .. of a 32-byte slice from thread t; a
// contraction may be taken in any order, so each thread's four words simply serve as (low, high) of two such slices, the
// same for both operands, and every load is one 16-byte access.
constexpr int kRowsWarps = 8;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int kTiles, typename OutT>
__global__ void __launch_bounds__(kRowsWarps * 32)
few_rows_kernel(const uint8_t* __restrict__ x, const float* __restrict__ x_scale, const uint8_t* __restrict__ w,
                const float* __restrict__ w_scale, OutT* __restrict__ out, long long ldd, int M, int N, int K) {
  constexpr int kUnroll = kTiles <= 2 ? 4 : 2;
  __shared__ float part[kRowsWarps][kTiles * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const bool ok0 = n0 + g < N, ok1 = n0 + g + 8 < N;
  const uint8_t* w0 = w + static_cast<long long>(n0 + g) * K;
  const uint8_t* w1 = w0 + 8LL * K;
  const uint8_t* xr = x + static_cast<long long>(g) * K;
  float acc[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k0 = warp * 64 + t * 16; k0 - t * 16 < K; k0 += kRowsWarps * 64 * kUnroll) {
    uint4 a0[kUnroll], a1[kUnroll], b[kUnroll][kTiles];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * kRowsWarps * 64;
      const bool in = k < K;  // K is a multiple of 16: a 16-byte piece is all in or all out
      a0[u] = in && ok0 ? __ldcs(reinterpret_cast<const uint4*>(w0 + k)) : zero;
      a1[u] = in && ok1 ? __ldcs(reinterpret_cast<const uint4*>(w1 + k)) : zero;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        b[u][i] = in && g + 8 * i < M ? __ldg(reinterpret_cast<const uint4*>(xr + 8LL * i * K + k)) : zero;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        mma_e4m3(acc[i], a0[u].x, a1[u].x, a0[u].y, a1[u].y, b[u][i].x, b[u][i].y);
        mma_e4m3(acc[i], a0[u].z, a1[u].z, a0[u].w, a1[u].w, b[u][i].z, b[u][i].w);
      }
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {  // accumulator: weight rows g, g + 8 x rows 2 t, 2 t + 1 of x
    part[warp][8 * i + 2 * t][g] = acc[i][0];
    part[warp][8 * i + 2 * t + 1][g] = acc[i][1];
    part[warp][8 * i + 2 * t][g + 8] = acc[i][2];
    part[warp][8 * i + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTiles * 8 * 16; i += kRowsWarps * 32) {
    const int m = i / 16, n = i % 16;
    if (m >= M || n0 + n >= N) continue;
    float s = part[0][m][n];
#pragma unroll
    for (int j = 1; j < kRowsWarps; ++j) s += part[j][m][n];
    s *= x_scale[m] * w_scale[n0 + n];
    if constexpr (sizeof(OutT) == 4) out[m * ldd + n0 + n] = s;
    else out[m * ldd + n0 + n] = __float2bfloat16_rn(s);
  }
}

constexpr int kFewRows = 32;

template <typename OutT>
int run_few_rows(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
                 cudaStream_t stream) {
  auto kern = M <= 8 ? few_rows_kernel<1, OutT> : M <= 16 ? few_rows_kernel<2, OutT> : few_rows_kernel<4, OutT>;
  kern<<<(N + 15) / 16, kRowsWarps * 32, 0, stream>>>(static_cast<const uint8_t*>(A), a_scale, static_cast<const uint8_t*>(B), b_scale,
                                                       static_cast<OutT*>(D), ldd, M, N, K);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string("e4m3 few-rows launch failed: ") + cudaGetErrorString(e));
  return kOk;
}

template <typename OutT>
int run_scaled(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
               int* dev_status, cudaStream_t stream) {
  if (M <= kFewRows) return run_few_rows<OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
  using Epi = EpiScaled<OutT>;
  const LaunchOptions opt = launch_options();
  if (opt.cta_group != 2) return fail(kBadArgument, "the e4m3 GEMM is built for CTA pairs only (cta_group = 2)");
  typename Epi::Params ep;
  ep.D = static_cast<OutT*>(D);
  ep.ldd = ldd;
  ep.row_scale = a_scale;
  ep.col_scale = b_scale;
  ep.use_tma = opt.epi_tma;
  const int rc = make_tmap_out(&ep.tm_d, ep.D, N, M, ldd);
  if (rc != kOk) return rc;
  const int K2 = K / 2;  // two e4m3 elements per two-byte unit
  switch (choose_tile_n(M, N, opt, true)) {
    case 64: return launch_gemm_cfg<2, 64, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
    case 128: return launch_gemm_cfg<2, 128, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
    default: return launch_gemm_cfg<2, 256, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
  }
}
}  // namespace

extern "C" int coda_b200_gemm_e4m3(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd,
                                   int d_is_fp32, int M, int N, int K, int* dev_status, void* stream) {
  if (!A || !a_scale || !B || !b_scale || !D) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || N <= 0 || K <= 0) return fail(kBadArgument, "GEMM extents must be positive");
  if (dev_status == nullptr) return fail(kBadArgument, "device status word is required");
  if (K % 16 != 0) return fail(kBadArgument, "K must be a multiple of 16");
  if (N % 8 != 0 || ldd % 8 != 0 || ldd < N) return fail(kBadArgument, "N and ldd must be multiples of 8 with ldd >= N");
  for (const void* p : {A, B, static_cast<const void*>(b_scale), static_cast<const void*>(D)})
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return fail(kBadArgument, "operands, output and column scales must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d_is_fp32) return run_scaled<float>(A, a_scale, B, b_scale, D, ldd, M, N, K, dev_status, st);
  return run_scaled<__nv_bfloat16>(A, a_scale, B, b_scale, D, ldd, M, N, K, dev_status, st);
}
