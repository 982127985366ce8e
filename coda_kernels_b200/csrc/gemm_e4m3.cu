// C-ABI entry point of the projection of e4m3 rows by an e4m3 weight.  See include/coda_b200.h for the contract.
#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// ------------------------------------------------------------------ few rows
// The product for a handful of rows of x is a stream of the weight through the SMs, bound by HBM: a tile of the GEMM core
// would keep 16 to 48 CTA pairs busy and fill most of its A operand with zeros.  Here a block owns 16 weight rows and its 8
// warps share out the contraction in steps of 64, four steps in flight; the warps' sums are added in shared memory in a fixed
// order.
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
__global__ void __launch_bounds__(kRowsWarps * 32, kTiles == 1 ? 4 : 1)
few_rows_kernel(const uint8_t* __restrict__ x, const float* __restrict__ x_scale, const uint8_t* __restrict__ w,
                const float* __restrict__ w_scale, OutT* __restrict__ out, long long ldd, int M, int N, int K) {
  constexpr int kUnroll = 4;
  __shared__ float part[kRowsWarps / 2][kTiles * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const uint8_t* wr = w + static_cast<long long>(n0 + g) * K;
  const uint8_t* xr = x + static_cast<long long>(g) * K;
  float acc[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k0 = warp * 64 + t * 16; k0 - t * 16 < K; k0 += kRowsWarps * 64 * kUnroll) {
    uint4 a[kUnroll][2], b[kUnroll][kTiles];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * kRowsWarps * 64;
      const bool in = k < K;  // K is a multiple of 16: a 16-byte piece is all in or all out
#pragma unroll
      for (int r = 0; r < 2; ++r)
        a[u][r] = in && n0 + g + 8 * r < N ? __ldcs(reinterpret_cast<const uint4*>(wr + 8LL * r * K + k)) : zero;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        b[u][i] = in && g + 8 * i < M ? __ldg(reinterpret_cast<const uint4*>(xr + 8LL * i * K + k)) : zero;
    }
    // all loads before the first product: left alone the compiler keeps fewer in flight (one row, 6144 x 4096: 9.3 instead of
    // 7.6 us)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        mma_e4m3(acc[i], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][i].x, b[u][i].y);
        mma_e4m3(acc[i], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][i].z, b[u][i].w);
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
        for (int j = 0; j < 4; ++j) part[warp - half][8 * i + 2 * t + (j & 1)][g + 8 * (j >> 1)] = acc[i][j];
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += part[warp][8 * i + 2 * t + (j & 1)][g + 8 * (j >> 1)];
    }
    __syncthreads();
  }
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[0][8 * i + 2 * t + (j & 1)][g + 8 * (j >> 1)] = acc[i][j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTiles * 8 * 16; i += kRowsWarps * 32) {
    const int m = i / 16, n = i % 16;
    if (m >= M || n0 + n >= N) continue;
    const float s = part[0][m][n] * (x_scale[m] * w_scale[n0 + n]);
    if constexpr (sizeof(OutT) == 4) out[m * ldd + n0 + n] = s;
    else out[m * ldd + n0 + n] = __float2bfloat16_rn(s);
  }
}

// Against the swapped tiles below, weights from HBM: to 8 rows 6144 x 4096 takes 7.6 us, 28672 x 4096 25 us and 4096 x 14336
// 17 us (swapped tiles, 17 rows: 14.5, 29 and 21 us); to 16 rows 11, 33 and 17 us.  Beyond, the blocks' reads of x weigh as much
// as the weight (32 rows: 15, 51 and 34 us in the best form tried).
constexpr int kFewRows = 16;

template <typename OutT>
int run_few_rows(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
                 cudaStream_t stream) {
  auto kern = M <= 8 ? few_rows_kernel<1, OutT> : few_rows_kernel<2, OutT>;
  kern<<<(N + 15) / 16, kRowsWarps * 32, 0, stream>>>(static_cast<const uint8_t*>(A), a_scale, static_cast<const uint8_t*>(B), b_scale,
                                                       static_cast<OutT*>(D), ldd, M, N, K);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string("e4m3 few-rows launch failed: ") + cudaGetErrorString(e));
  return kOk;
}

// ------------------------------------------------------------------ up to kSwapRows rows
// With so few rows of x the GEMM core's 256-row tile would load mostly padding, and there would be too few column tiles for
// the SMs.  So the weight takes the rows' place (256 of them a tile, whole) and x the columns', in the narrowest tile that
// holds it; the tiles of the last round, which here is often the only one, are cut along K.  Weights from HBM, 32 and 64 rows:
// 6144 x 4096 14.6 and 15.4 us (not swapped 17.8), 28672 x 4096 29 and 30 us (35), 4096 x 14336 21 and 22 us (39).  To 128 rows the
// parts cost as much as they save unless the contraction is long: 4096 x 4096 18.5 us (16.1), 4096 x 14336 26 us (39).
constexpr int kSwapRows = 128;
inline bool swapped(int M, int K) { return M > kFewRows && (M <= 64 || (M <= kSwapRows && K >= 8192)); }

// Adds the parts of the cut tiles in order, scales them, and writes the transposed tile: block (t, b) has 32 accumulator rows
// of tail tile t, which it turns through shared memory.
template <typename OutT>
__global__ void __launch_bounds__(256) scaled_finalize_kernel(const float* __restrict__ ws, OutT* __restrict__ D, long long ldd,
                                                              GemmShape shape, int first_tail_tile, int tile_m, int bn,
                                                              const float* __restrict__ row_scale, const float* __restrict__ col_scale) {
  __shared__ float turned[32][kSwapRows + 1];
  int tm, tn;
  tile_coords(shape, first_tail_tile + static_cast<int>(blockIdx.x), tm, tn);
  const int r0 = blockIdx.y * 32, row0 = tm * tile_m + r0, groups = bn / 4;
  const long long slab = static_cast<long long>(tile_m) * bn;
  for (int i = threadIdx.x; i < 32 * groups; i += 256) {
    const int r = i / groups, g = i % groups;
    const float* src = ws + blockIdx.x * slab + static_cast<long long>(r0 + r) * bn + g * 4;
    float4 acc = __ldcs(reinterpret_cast<const float4*>(src));
#pragma unroll 4
    for (int part = 1; part < shape.sk_split; ++part) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src + static_cast<long long>(part) * shape.sk_tail * slab));
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
    turned[r][4 * g] = acc.x;
    turned[r][4 * g + 1] = acc.y;
    turned[r][4 * g + 2] = acc.z;
    turned[r][4 * g + 3] = acc.w;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, row = row0 + lane;
  if (row >= shape.M) return;
  const float rs = row_scale[row];
  for (int c = threadIdx.x / 32; c < bn; c += 8) {
    const int col = tn * bn + c;
    if (col >= shape.N) break;
    const float v = turned[lane][c] * (rs * col_scale[col]);
    if constexpr (sizeof(OutT) == 4) D[col * ldd + row] = v;
    else D[col * ldd + row] = __float2bfloat16_rn(v);
  }
}

inline int swap_tile_n(int M) { return M <= 64 ? 64 : 128; }

template <typename OutT>
int run_swapped(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
                void* workspace, int64_t workspace_bytes, int* dev_status, cudaStream_t stream, const LaunchOptions& opt) {
  using Epi = EpiScaledT<OutT>;
  typename Epi::Params ep;
  memset(&ep.tm_ws, 0, sizeof(ep.tm_ws));
  ep.D = static_cast<OutT*>(D);
  ep.ldd = ldd;
  ep.row_scale = b_scale;
  ep.col_scale = a_scale;
  ep.ws = static_cast<float*>(workspace);
  ep.ws_bytes = workspace_bytes;
  const int K2 = K / 2;
  if (swap_tile_n(M) == 64)
    return launch_gemm_cfg<2, 64, false, false, Epi, ProE4M3>(B, K2, A, K2, N, M, K2, ep, dev_status, stream, opt);
  return launch_gemm_cfg<2, 128, false, false, Epi, ProE4M3>(B, K2, A, K2, N, M, K2, ep, dev_status, stream, opt);
}

}  // namespace

namespace cb {
template <typename OutT>
struct SplitFinalize<EpiScaledT<OutT>> {
  static void launch(const typename EpiScaledT<OutT>::Params& ep, const GemmShape& shape, int first_tail_tile, int tile_m, int bn,
                     cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(shape.sk_tail), static_cast<unsigned>(tile_m / 32), 1);
    scaled_finalize_kernel<OutT><<<grid, 256, 0, stream>>>(ep.ws, ep.D, ep.ldd, shape, first_tail_tile, tile_m, bn, ep.row_scale, ep.col_scale);
  }
};
}  // namespace cb

namespace {

// The narrowest tile whose tiles all run at once, so that as many SMs as possible share the work; otherwise as for the other
// GEMMs (333 x 2056 x 1552: 9.7 us with 64 columns, 10.7 with 128, 13.8 with 256).
inline int tile_n(int M, int N, const LaunchOptions& opt) {
  const long long tiles_m = (M + 2 * kBlockM - 1) / (2 * kBlockM), clusters = full_clusters(opt, 2);
  for (int bn = 64; bn < 256 && opt.tile_n == 0; bn *= 2)
    if (tiles_m * ((N + bn - 1) / bn) <= clusters) return bn;
  return choose_tile_n(M, N, opt, true);
}

template <typename OutT>
int run_scaled(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
               void* workspace, int64_t workspace_bytes, int* dev_status, cudaStream_t stream) {
  if (M <= kFewRows) return run_few_rows<OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, stream);
  using Epi = EpiScaled<OutT>;
  const LaunchOptions opt = launch_options();
  if (opt.cta_group != 2) return fail(kBadArgument, "the e4m3 GEMM is built for CTA pairs only (cta_group = 2)");
  if (swapped(M, K)) return run_swapped<OutT>(A, a_scale, B, b_scale, D, ldd, M, N, K, workspace, workspace_bytes, dev_status, stream, opt);
  typename Epi::Params ep;
  ep.D = static_cast<OutT*>(D);
  ep.ldd = ldd;
  ep.row_scale = a_scale;
  ep.col_scale = b_scale;
  ep.use_tma = opt.epi_tma;
  const int rc = make_tmap_out(&ep.tm_d, ep.D, N, M, ldd);
  if (rc != kOk) return rc;
  const int K2 = K / 2;  // two e4m3 elements per two-byte unit
  switch (tile_n(M, N, opt)) {
    case 64: return launch_gemm_cfg<2, 64, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
    case 128: return launch_gemm_cfg<2, 128, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
    default: return launch_gemm_cfg<2, 256, false, false, Epi, ProE4M3>(A, K2, B, K2, M, N, K2, ep, dev_status, stream, opt);
  }
}
}  // namespace

extern "C" int64_t coda_b200_gemm_e4m3_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || !swapped(M, K)) return 0;
  const LaunchOptions opt = launch_options();
  if (opt.split_tail == 0 || opt.cta_group != 2) return 0;
  const int clusters = full_clusters(opt, 2);
  int tail = 0;
  if (plan_tail_split((N + 2 * kBlockM - 1) / (2 * kBlockM), (K / 2 + kBlockK - 1) / kBlockK, clusters, &tail) <= 1) return 0;
  return split_workspace_bytes(clusters, 2 * kBlockM, swap_tile_n(M));
}

extern "C" int coda_b200_gemm_e4m3(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd,
                                   int d_is_fp32, int M, int N, int K, void* workspace, int64_t workspace_bytes, int* dev_status,
                                   void* stream) {
  if (!A || !a_scale || !B || !b_scale || !D) return fail(kBadArgument, "NULL pointer");
  if (M <= 0 || N <= 0 || K <= 0) return fail(kBadArgument, "GEMM extents must be positive");
  if (M > 1 << 30 || N > 1 << 30 || K > 1 << 30) return fail(kBadArgument, "GEMM extents must not exceed 2^30");
  if (dev_status == nullptr) return fail(kBadArgument, "device status word is required");
  if (K % 16 != 0) return fail(kBadArgument, "K must be a multiple of 16");
  if (N % 8 != 0 || ldd % 8 != 0 || ldd < N) return fail(kBadArgument, "N and ldd must be multiples of 8 with ldd >= N");
  if (workspace_bytes < 0) return fail(kBadArgument, "workspace_bytes must not be negative");
  for (const void* p : {A, B, static_cast<const void*>(D), static_cast<const void*>(workspace)})
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return fail(kBadArgument, "operands, output and workspace must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d_is_fp32) return run_scaled<float>(A, a_scale, B, b_scale, D, ldd, M, N, K, workspace, workspace_bytes, dev_status, st);
  return run_scaled<__nv_bfloat16>(A, a_scale, B, b_scale, D, ldd, M, N, K, workspace, workspace_bytes, dev_status, st);
}
