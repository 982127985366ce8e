// Row kernels around the fused linears: counter-based dropout, the residual addition with dropout and RMS norm
// (forward and backward), and rows leaving as e4m3 values with one scale each.  Matrices are dense [rows, cols] of
// bf16, fp16 or fp32; all arithmetic is fp32.  See include/coda_b200.h for the contract.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

constexpr int kRowThreads = 256;

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// ------------------------------------------------------------------ dropout mask
// Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
// Key = seed; counter = (block, step, stream); the four words of block r * ceil(cols / 4) + c / 4 decide elements
// c .. c + 3 of row r.  An element stays if its word is >= threshold = round(p * 2^32).
struct Dropout {
  const long long* rng;  // device [seed, step]; nullptr: nothing is dropped
  uint32_t stream, threshold;
  float scale;  // 1 / (1 - p)
};

struct Mask {
  uint32_t k0, k1, step, stream, threshold;

  __device__ explicit Mask(const Dropout& d) : k0(0), k1(0), step(0), stream(d.stream), threshold(d.threshold) {
    if (d.rng != nullptr) {
      const unsigned long long seed = static_cast<unsigned long long>(__ldg(d.rng));
      k0 = static_cast<uint32_t>(seed);
      k1 = static_cast<uint32_t>(seed >> 32);
      step = static_cast<uint32_t>(__ldg(d.rng + 1));
    }
  }
  __device__ uint4 words(unsigned long long block) const {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = step, c3 = stream, a = k0, b = k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const unsigned long long p0 = static_cast<unsigned long long>(c0) * 0xD2511F53u;
      const unsigned long long p1 = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
      c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ a;
      c1 = static_cast<uint32_t>(p1);
      c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ b;
      c3 = static_cast<uint32_t>(p0);
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
  // v of element `col` of `row` after dropout: a dropped value is +0 whatever it held
  __device__ float apply(float v, long long row, int col, int blocks, float scale) const {
    const uint4 w = words(static_cast<unsigned long long>(row) * blocks + (col >> 2));
    const int j = col & 3;
    const uint32_t u = j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w;
    return u >= threshold ? v * scale : 0.0f;
  }
};

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // the previous use of red is over
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) s += red[i];
  return s;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) s = max_nan(s, red[i]);
  return s;
}

// ------------------------------------------------------------------ dropout alone
template <typename T>
__global__ void __launch_bounds__(kRowThreads) dropout_kernel(const T* __restrict__ x, T* __restrict__ out, long long rows, int cols,
                                                              Dropout d, long long* __restrict__ used) {
  const Mask mask(d);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
  const int blocks = (cols + 3) / 4;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += kRowThreads) {
      const float v = to_f32(x[row * cols + c]);
      out[row * cols + c] = from_f32<T>(d.rng != nullptr ? mask.apply(v, row, c, blocks, d.scale) : v);
    }
}

// ------------------------------------------------------------------ residual + dropout(x), RMS norm
// One block per row.  h = residual + dropout(x) (x alone without a residual); rstd = rsqrt(mean(h^2) + eps), taken of
// the unrounded h; out = h * rstd * w.  kE4M3: out leaves as e4m3 values q with scale = max(max|out| / 448, 2^-126),
// q = out / scale rounded once; without a weight the rows are converted as they are.
template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kRowThreads) norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                               const T* __restrict__ weight, float eps, Dropout d,
                                                               long long* __restrict__ used, T* __restrict__ h, T* __restrict__ out,
                                                               float* __restrict__ rstd, __nv_fp8_e4m3* __restrict__ q,
                                                               float* __restrict__ scale, long long rows, int cols) {
  __shared__ float red[kRowThreads / 32];
  const Mask mask(d);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
  const int blocks = (cols + 3) / 4;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long long base = row * cols;
    auto value = [&](int c) {
      float v = to_f32(x[base + c]);
      if (d.rng != nullptr) v = mask.apply(v, row, c, blocks, d.scale);
      return residual != nullptr ? v + to_f32(residual[base + c]) : v;
    };
    float sq = 0.f, top = 0.f;
    for (int c = threadIdx.x; c < cols; c += kRowThreads) {
      const float v = value(c);
      if (h != nullptr) h[base + c] = from_f32<T>(v);
      sq = fmaf(v, v, sq);
      if (kE4M3) top = max_nan(top, fabsf(weight != nullptr ? v * to_f32(weight[c]) : v));
    }
    const float r = weight != nullptr ? rsqrtf(block_sum(sq, red) / static_cast<float>(cols) + eps) : 1.0f;
    float s = 1.0f;
    if (kE4M3) {
      s = max_nan(block_max(top, red) * r / 448.0f, 1.17549435e-38f);
      if (threadIdx.x == 0) scale[row] = s;
    } else if (threadIdx.x == 0) {
      rstd[row] = r;
    }
    for (int c = threadIdx.x; c < cols; c += kRowThreads) {
      const float v = value(c);
      const float o = weight != nullptr ? v * r * to_f32(weight[c]) : v;
      if (kE4M3) q[base + c] = __nv_fp8_e4m3(o / s);
      else out[base + c] = from_f32<T>(o);
    }
  }
}

// ------------------------------------------------------------------ its backward
// g = dout * w, xh = h * rstd, c = mean(g * xh): dres = dh + rstd * (g - xh * c), dx = dropout(dres), and one partial row
// of sum(dout * xh) a block.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ dh, const T* __restrict__ h,
                                                               const float* __restrict__ rstd, const T* __restrict__ weight, Dropout d,
                                                               T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partial,
                                                               long long rows, int cols) {
  __shared__ float red[kRowThreads / 32];
  const Mask mask(d);
  const int blocks = (cols + 3) / 4;
  float* mine = partial != nullptr ? partial + static_cast<long long>(blockIdx.x) * cols : nullptr;
  if (mine != nullptr)
    for (int c = threadIdx.x; c < cols; c += kRowThreads) mine[c] = 0.f;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long long base = row * cols;
    const float r = rstd[row];
    float dot = 0.f;
    for (int c = threadIdx.x; c < cols; c += kRowThreads) {
      const float o = to_f32(dout[base + c]), xh = to_f32(h[base + c]) * r;
      dot = fmaf(o * to_f32(weight[c]), xh, dot);
      if (mine != nullptr) mine[c] += o * xh;
    }
    const float m = block_sum(dot, red) / static_cast<float>(cols);
    for (int c = threadIdx.x; c < cols; c += kRowThreads) {
      const float g = to_f32(dout[base + c]) * to_f32(weight[c]), xh = to_f32(h[base + c]) * r;
      float v = r * (g - xh * m);
      if (dh != nullptr) v += to_f32(dh[base + c]);
      if (dres != nullptr) dres[base + c] = from_f32<T>(v);
      if (dx != nullptr) dx[base + c] = from_f32<T>(d.rng != nullptr ? mask.apply(v, row, c, blocks, d.scale) : v);
    }
  }
}

// Column sums of the partial rows, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) fold_rows_kernel(const float* __restrict__ partial, int nrows, int cols, T* __restrict__ out) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int b = ry; b < nrows; b += 32) s += partial[static_cast<long long>(b) * cols + c];
  }
  red[ry][cx] = s;
  __syncthreads();
  if (ry == 0 && c < cols) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) t += red[j][cx];
    out[c] = from_f32<T>(t);
  }
}

// ------------------------------------------------------------------ host side
inline int launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(kCudaError, std::string(what) + ": " + cudaGetErrorString(e));
  return kOk;
}

inline int check_extents(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0 || cols <= 0 || cols > 0x7ffffff0LL) return fail(kBadArgument, "rows must not be negative and cols must be positive (and fit 31 bits)");
  if (dtype < 0 || dtype > 2) return fail(kBadArgument, "dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  return kOk;
}

inline int make_dropout(double p, const int64_t* rng, int64_t stream_id, Dropout* d) {
  if (!(p >= 0.0 && p < 1.0)) return fail(kBadArgument, "dropout probability must be at least 0 and below 1");
  if (stream_id < 0 || stream_id > 0xffffffffLL) return fail(kBadArgument, "dropout stream must fit 32 bits");
  if (p > 0.0 && rng == nullptr) return fail(kBadArgument, "dropout needs the generator's [seed, step]");
  d->rng = p > 0.0 ? reinterpret_cast<const long long*>(rng) : nullptr;
  d->stream = static_cast<uint32_t>(stream_id);
  const double t = std::nearbyint(p * 4294967296.0);
  d->threshold = t >= 4294967295.0 ? 0xffffffffu : static_cast<uint32_t>(t);
  d->scale = static_cast<float>(1.0 / (1.0 - p));
  return kOk;
}

inline int row_grid(int64_t rows) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<int>(rows < cap ? rows : cap);
}
inline int64_t bwd_blocks(int64_t rows) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * 4;
  return rows < cap ? rows : cap;
}

template <class F>
int by_dtype(int dtype, F&& f) {
  if (dtype == 0) return f(__nv_bfloat16());
  if (dtype == 1) return f(__half());
  return f(float());
}

}  // namespace

extern "C" int coda_b200_dropout(const void* x, void* out, int64_t rows, int64_t cols, int dtype, double p, const int64_t* rng,
                                 int64_t stream_id, int64_t* rng_used, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !out) return fail(kBadArgument, "NULL pointer");
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    dropout_kernel<T><<<row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(x), static_cast<T*>(out), rows, static_cast<int>(cols), d, reinterpret_cast<long long*>(rng_used));
    return launch_check("dropout launch");
  });
}

extern "C" int coda_b200_add_rmsnorm_fwd(const void* x, const void* residual, const void* weight, float eps, double p, const int64_t* rng,
                                         int64_t stream_id, int64_t* rng_used, void* h, void* out, float* rstd, int64_t rows,
                                         int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !weight || !out || !rstd) return fail(kBadArgument, "NULL pointer");
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    norm_fwd_kernel<T, false><<<row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), eps, d,
        reinterpret_cast<long long*>(rng_used), static_cast<T*>(h), static_cast<T*>(out), rstd, nullptr, nullptr, rows,
        static_cast<int>(cols));
    return launch_check("add_rmsnorm forward launch");
  });
}

extern "C" int coda_b200_rows_e4m3(const void* x, const void* residual, const void* weight, float eps, void* h, void* q, float* scale,
                                   int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !q || !scale) return fail(kBadArgument, "NULL pointer");
  const Dropout d{nullptr, 0u, 0u, 1.0f};
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    norm_fwd_kernel<T, true><<<row_grid(rows), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), eps, d, nullptr, static_cast<T*>(h),
        nullptr, nullptr, static_cast<__nv_fp8_e4m3*>(q), scale, rows, static_cast<int>(cols));
    return launch_check("e4m3 rows launch");
  });
}

extern "C" int64_t coda_b200_add_rmsnorm_bwd_scratch_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : bwd_blocks(rows) * cols * static_cast<int64_t>(sizeof(float));
}

extern "C" int coda_b200_add_rmsnorm_bwd(const void* dout, const void* dh, const void* h, const float* rstd, const void* weight, double p,
                                         const int64_t* rng, int64_t stream_id, void* dx, void* dres, void* dweight, void* scratch,
                                         int64_t scratch_bytes, int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!dout || !h || !rstd || !weight) return fail(kBadArgument, "NULL pointer");
  if (dweight != nullptr && (scratch == nullptr || scratch_bytes < coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols)))
    return fail(kBadArgument, "the weight gradient needs coda_b200_add_rmsnorm_bwd_scratch_bytes of scratch");
  const int blocks = static_cast<int>(bwd_blocks(rows)), n = static_cast<int>(cols);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    norm_bwd_kernel<T><<<blocks, kRowThreads, 0, st>>>(static_cast<const T*>(dout), static_cast<const T*>(dh), static_cast<const T*>(h), rstd,
                                                       static_cast<const T*>(weight), d, static_cast<T*>(dx), static_cast<T*>(dres),
                                                       dweight != nullptr ? static_cast<float*>(scratch) : nullptr, rows, n);
    int rc2 = launch_check("add_rmsnorm backward launch");
    if (rc2 != kOk || dweight == nullptr) return rc2;
    fold_rows_kernel<T><<<(n + 31) / 32, 1024, 0, st>>>(static_cast<const float*>(scratch), blocks, n, static_cast<T*>(dweight));
    return launch_check("add_rmsnorm weight gradient launch");
  });
}
