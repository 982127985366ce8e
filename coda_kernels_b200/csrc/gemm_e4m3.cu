// C-ABI entry point of the projection of e4m3 rows by an e4m3 weight.  See include/coda_b200.h for the contract.
#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {
template <typename OutT>
int run_scaled(const void* A, const float* a_scale, const void* B, const float* b_scale, void* D, int64_t ldd, int M, int N, int K,
               int* dev_status, cudaStream_t stream) {
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
