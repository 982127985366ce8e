// C-ABI entry point of the projection of e4m3 rows by an e4m3 weight.  See include/coda_b200.h for the contract.
#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// ------------------------------------------------------------------ few rows
// The product for a handful of rows of x is a stream of the weight through the SMs, bound by HBM: a tile of the GEMM core
// would keep 16 to 48 CTA pairs busy and fill most of its A operand with zeros.  Here a block owns 16 * kBands weight rows
// and its 8 warps share out the contraction in steps of 64; the warps' sums are added in shared memory in a fixed order.
//
// The product itself is mma.sync m16n8k32 with the weight rows as M and the rows of x as N (kTiles tiles of 8).  A thread
// holds, for weight rows g and g + 8 (g = lane / 4), 16 consecutive bytes at 16 (lane % 4) of the step, and the same 16
// bytes of row g of x.  The instruction wants bytes 4 t .. 4 t + 3 and 16 + 4 t .. of a 32-byte slice from thread t; a
// contraction may be taken in any order, so each thread's four words simply serve as (low, high) of two such slices, the
// same for both operands, and every load is one 16-byte access.
//
// Every block reads all of x, mostly from L2, so beyond 16 rows it takes two bands of weight rows (kBands).
constexpr int kRowsWarps = 8;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int kTiles, int kBands, int kUnroll, typename OutT>
__global__ void __launch_bounds__(kRowsWarps * 32, kTiles == 1 ? 4 : 1)
few_rows_kernel(const uint8_t* __restrict__ x, const float* __restrict__ x_scale, const uint8_t* __restrict__ w,
                const float* __restrict__ w_scale, OutT* __restrict__ out, long long ldd, int M, int N, int K) {
  constexpr int kCols = 16 * kBands;
  __shared__ float part[kRowsWarps / 2][kTiles * 8][kCols + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kCols;
  const uint8_t* wr = w + static_cast<long long>(n0 + g) * K;
  const uint8_t* xr = x + static_cast<long long>(g) * K;
  float acc[kBands][kTiles][4];
#pragma unroll
  for (int r = 0; r < kBands; ++r)
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[r][i][0] = acc[r][i][1] = acc[r][i][2] = acc[r][i][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k0 = warp * 64 + t * 16; k0 - t * 16 < K; k0 += kRowsWarps * 64 * kUnroll) {
    uint4 a[kUnroll][2 * kBands], b[kUnroll][kTiles];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * kRowsWarps * 64;
      const bool in = k < K;  // K is a multiple of 16: a 16-byte piece is all in or all out
#pragma unroll
      for (int r = 0; r < 2 * kBands; ++r)
        a[u][r] = in && n0 + g + 8 * r < N ? __ldcs(reinterpret_cast<const uint4*>(wr + 8LL * r * K + k)) : zero;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        b[u][i] = in && g + 8 * i < M ? __ldg(reinterpret_cast<const uint4*>(xr + 8LL * i * K + k)) : zero;
    }
    // all loads before the first product: left alone the compiler keeps fewer in flight (one row, 6144 x 4096: 9.3 instead of
    // 7.6 us); with four tiles it is the other way round (22 instead of 15 us)
    if constexpr (kTiles <= 2) asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int r = 0; r < kBands; ++r) {
          mma_e4m3(acc[r][i], a[u][2 * r].x, a[u][2 * r + 1].x, a[u][2 * r].y, a[u][2 * r + 1].y, b[u][i].x, b[u][i].y);
          mma_e4m3(acc[r][i], a[u][2 * r].z, a[u][2 * r + 1].z, a[u][2 * r].w, a[u][2 * r + 1].w, b[u][i].z, b[u][i].w);
        }
  }
  // accumulator: weight rows g, g + 8 x rows 2 t, 2 t + 1 of x.  The upper half of the warps hands its sums to the lower
  // half until one is left.
#pragma unroll
  for (int half = kRowsWarps / 2; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int r = 0; r < kBands; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[warp - half][8 * i + 2 * t + (j & 1)][16 * r + g + 8 * (j >> 1)] = acc[r][i][j];
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int r = 0; r < kBands; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[r][i][j] += part[warp][8 * i + 2 * t + (j & 1)][16 * r + g + 8 * (j >> 1)];
    }
    __syncthreads();
  }
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int r = 0; r < kBands; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[0][8 * i + 2 * t + (j & 1)][16 * r + g + 8 * (j >> 1)] = acc[r][i][j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTiles * 8 * kCols; i += kRowsWarps * 32) {
    const int m = i / kCols, n = i % kCols;
    if (m >= M || n0 + n >= N) continue;
    const float s = part[0][m][n] * (x_scale[m] * w_scale[n0 + n]);
    if constexpr (sizeof(OutT) == 4) out[m * ldd + n0 + n] = s;
    else out[m * ldd + n0 + n] = __float2bfloat16_rn(s);
  }
}

// Against the GEMM core's tiles, weights from HBM: 28672 x 4096 takes 25 us to 8 rows and 33 us to 16, where the tiles take 37 us
// for any count to 128; 6144 x 4096 7.6 and 11 us, the tiles 19 us.  From 17 rows on the blocks' reads of x weigh as much as
// the weight: 4096 x 4096 to 32 rows 12 us, the tiles 18 us; but 6144 x 4096, whose blocks no longer run at once, 22 us.
inline bool few_rows(int M, int N) { return M <= 16 || (M <= 32 && (N + 31) / 32 <= sm_count()); }

template <int kTiles, int kBands, int kUnroll, typename OutT>
int launch_few_rows(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
                    cudaStream_t stream) {
  few_rows_kernel<kTiles, kBands, kUnroll, OutT><<<(N + 16 * kBands - 1) / (16 * kBands), kRowsWarps * 32, 0, stream>>>(
      static_cast<const uint8_t*>(A), a_scale, static_cast<const uint8_t*>(B), b_scale, static_cast<OutT*>(D), ldd, M, N, K);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string("e4m3 few-rows launch failed: ") + cudaGetErrorString(e));
  return kOk;
}
template <typename OutT>
int run_few_rows(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
                 cudaStream_t stream) {
  if (M <= 8) return launch_few_rows<1, 1, 4, OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
  if (M <= 16) return launch_few_rows<2, 1, 4, OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
  return launch_few_rows<4, 2, 1, OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
}

template <typename OutT>
int run_scaled(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
               int* dev_status, cudaStream_t stream) {
  if (few_rows(M, N)) return run_few_rows<OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
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
