// Row kernels around the fused linears: counter-based dropout, the residual addition with dropout and RMS norm
// (forward and backward), and rows leaving as e4m3 values with one scale each.  Matrices are dense [rows, cols] of
// bf16, fp16 or fp32; all arithmetic is fp32.  See include/coda_b200.h for the contract.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <type_traits>

#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// ------------------------------------------------------------------ chunks
// A thread works on chunks of 8 consecutive elements of a row, held as loaded (2-byte types: 4 registers, fp32: 8).
// kVec: every chunk is whole and 16-byte aligned, and moves in 16-byte accesses; otherwise `n` elements (which may be <= 0)
// move one by one.  Elements that are not there read as zero.
template <typename T>
struct Chunk {
  uint32_t w[2 * sizeof(T)];
};
__device__ __forceinline__ float chunk_get(const Chunk<__nv_bfloat16>& c, int i) {
  return __uint_as_float((i & 1) ? (c.w[i >> 1] & 0xffff0000u) : (c.w[i >> 1] << 16));
}
__device__ __forceinline__ float chunk_get(const Chunk<__half>& c, int i) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? (c.w[i >> 1] >> 16) : c.w[i >> 1])));
}
__device__ __forceinline__ float chunk_get(const Chunk<float>& c, int i) { return __uint_as_float(c.w[i]); }

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

template <bool kVec, typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p, int n) {
  Chunk<T> c;
  if constexpr (kVec) {
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (n > 0) u = *(reinterpret_cast<const uint4*>(p) + k);
      c.w[4 * k] = u.x;
      c.w[4 * k + 1] = u.y;
      c.w[4 * k + 2] = u.z;
      c.w[4 * k + 3] = u.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c.w[j] = j < n ? __float_as_uint(p[j]) : 0u;
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
    unsigned short e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < n ? q[j] : static_cast<unsigned short>(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) c.w[j] = static_cast<uint32_t>(e[2 * j]) | (static_cast<uint32_t>(e[2 * j + 1]) << 16);
  }
  return c;
}
template <bool kVec, typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* v, int n) {
  if constexpr (!kVec) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = from_f32<T>(v[j]);
  } else if (n > 0) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
  }
}

// v * inv as e4m3.  inv is the row's 1 / scale: a division for every element made this kernel slower than its memory traffic
// (8192 x 5120 bf16: 125 us a pass with, 72 us without); the product's extra rounding of 2^-24 moves a value only where it lies
// that near to the middle of two e4m3 values.  Saturation turns 448 (1 + 2^-23) into 448.
template <bool kVec>
__device__ __forceinline__ void store_e4m3(__nv_fp8_e4m3* p, const float* v, float inv, int n) {
  uint32_t e[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) e[j] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * j] * inv, v[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  if constexpr (kVec) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j].__x = static_cast<__nv_fp8_storage_t>(e[j / 2] >> (8 * (j & 1)));
  }
}

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
  uint32_t key[20];  // the ten rounds' two key words
  uint32_t step, stream, threshold;
  float scale;

  __device__ explicit Mask(const Dropout& d) : step(0), stream(d.stream), threshold(d.threshold), scale(d.scale) {
    uint32_t k0 = 0, k1 = 0;
    if (d.rng != nullptr) {
      const unsigned long long seed = static_cast<unsigned long long>(__ldg(d.rng));
      k0 = static_cast<uint32_t>(seed);
      k1 = static_cast<uint32_t>(seed >> 32);
      step = static_cast<uint32_t>(__ldg(d.rng + 1));
    }
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      key[2 * i] = k0 + i * 0x9E3779B9u;
      key[2 * i + 1] = k1 + i * 0xBB67AE85u;
    }
  }
  __device__ __forceinline__ uint4 words(unsigned long long block) const {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = step, c3 = stream;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const unsigned long long p0 = static_cast<unsigned long long>(c0) * 0xD2511F53u;
      const unsigned long long p1 = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
      c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ key[2 * i];
      c1 = static_cast<uint32_t>(p1);
      c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ key[2 * i + 1];
      c3 = static_cast<uint32_t>(p0);
    }
    return make_uint4(c0, c1, c2, c3);
  }
  // the 8 values of a chunk whose first generator block is `block`, after dropout: a dropped value is +0 whatever it held
  __device__ __forceinline__ void apply(float* v, unsigned long long block) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint4 u = words(block + k);
      v[4 * k] = u.x >= threshold ? v[4 * k] * scale : 0.0f;
      v[4 * k + 1] = u.y >= threshold ? v[4 * k + 1] * scale : 0.0f;
      v[4 * k + 2] = u.z >= threshold ? v[4 * k + 2] * scale : 0.0f;
      v[4 * k + 3] = u.w >= threshold ? v[4 * k + 3] * scale : 0.0f;
    }
  }
};

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// (sum of a, max of b) over the kGroup threads of a row: a warp, or the whole block
template <int kGroup, bool kMax>
__device__ __forceinline__ void row_reduce(float& a, float& b, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    if (kMax) b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
  if constexpr (kGroup > 32) {
    constexpr int kWarps = kGroup / 32;
    __syncthreads();  // the previous use of red is over
    if ((threadIdx.x & 31) == 0) {
      red[threadIdx.x >> 5] = a;
      if (kMax) red[kWarps + (threadIdx.x >> 5)] = b;
    }
    __syncthreads();
    a = red[0];
    if (kMax) b = red[kWarps];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
      a += red[i];
      if (kMax) b = max_nan(b, red[kWarps + i]);
    }
  }
}

// ------------------------------------------------------------------ dropout alone
// A stream of chunks, kDropUnroll of them in flight a thread.  Rows whose length is a multiple of 4 are one long row (the
// generator's blocks do not care), so `cols` may exceed 31 bits here.
constexpr int kDropThreads = 256, kDropUnroll = 2;
template <typename T, bool kVec>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const T* __restrict__ x, T* __restrict__ out, long long rows, long long cols,
                                                               Dropout d, long long* __restrict__ used) {
  const Mask mask(d);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
  const bool drop = d.rng != nullptr;
  const long long per_row = (cols + 7) / 8, blocks = (cols + 3) / 4, total = rows * per_row;
  const long long stride = static_cast<long long>(gridDim.x) * kDropThreads;
  for (long long i0 = blockIdx.x * static_cast<long long>(kDropThreads) + threadIdx.x; i0 < total; i0 += stride * kDropUnroll) {
    Chunk<T> in[kDropUnroll];
    long long at[kDropUnroll], block[kDropUnroll];
    int n[kDropUnroll];
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const long long i = i0 + k * stride;
      const long long row = rows == 1 ? 0 : i / per_row, c = 8 * (i - row * per_row);
      n[k] = i < total ? static_cast<int>(cols - c < 8 ? cols - c : 8) : 0;
      at[k] = row * cols + c;
      block[k] = row * blocks + c / 4;
      in[k] = load_chunk<kVec>(x + at[k], n[k]);
    }
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      if (n[k] <= 0) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = chunk_get(in[k], j);
      if (drop) mask.apply(v, block[k]);
      store_chunk<kVec>(out + at[k], v, n[k]);
    }
  }
}

// ------------------------------------------------------------------ residual + dropout(x), RMS norm
// h = residual + dropout(x) (x alone without a residual); rstd = rsqrt(mean(h^2) + eps), taken of the unrounded h; out =
// h * rstd * w.  kE4M3: out leaves as e4m3 values q with scale = max(max|out| / 448, 2^-126), q = out / scale rounded
// once; without a weight the rows are converted as they are.
//
// Bound by HBM.  kGroup threads own a row (a warp: kGroup = 32, several rows a block; else the block) and keep its h in
// registers as kChunks chunks each, so every tensor is read or written once; row_reduce is the only synchronisation.
template <typename T, bool kVec, int kGroup, int kChunks, bool kE4M3>
__global__ void __launch_bounds__(kGroup < 256 ? 256 : kGroup)
norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ weight, float eps, Dropout d,
                long long* __restrict__ used, T* __restrict__ h, T* __restrict__ out, float* __restrict__ rstd,
                __nv_fp8_e4m3* __restrict__ q, float* __restrict__ scale, long long rows, int cols) {
  __shared__ float red[2 * 32];
  const Mask mask(d);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
  const bool drop = d.rng != nullptr;
  const int blocks = (cols + 3) / 4;
  const int lane = kGroup == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int per_block = kGroup == 32 ? blockDim.x / 32 : 1;
  for (long long row = static_cast<long long>(blockIdx.x) * per_block + (kGroup == 32 ? threadIdx.x / 32 : 0); row < rows;
       row += static_cast<long long>(gridDim.x) * per_block) {
    const long long base = row * cols;
    float v[kChunks][8];
    Chunk<T> a[kChunks], b[kChunks];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
      a[k] = load_chunk<kVec>(x + base + c, n);
      if (residual != nullptr) b[k] = load_chunk<kVec>(residual + base + c, n);
    }
    float sq = 0.f, top = 0.f;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = chunk_get(a[k], j);
      if (drop && n > 0) mask.apply(v[k], static_cast<unsigned long long>(row) * blocks + c / 4);
      if (residual != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] += chunk_get(b[k], j);
      }
      if (h != nullptr) store_chunk<kVec>(h + base + c, v[k], n);
      // (elements past the row are zero: x reads as zero there and dropout keeps zeros)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[k][j], v[k][j], sq);
      if (kE4M3) {
        if (weight != nullptr) {
          const Chunk<T> w = load_chunk<kVec>(weight + c, n);
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(v[k][j] * chunk_get(w, j)));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(v[k][j]));
        }
      }
    }
    row_reduce<kGroup, kE4M3>(sq, top, red);
    const float r = weight != nullptr ? rsqrtf(sq / static_cast<float>(cols) + eps) : 1.0f;
    float s = 1.0f;
    if (kE4M3) s = max_nan(top * r / 448.0f, 1.17549435e-38f);
    const float inv = 1.0f / s;
    if (lane == 0) {
      if (kE4M3) scale[row] = s;
      else rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
      if (weight != nullptr) {
        const Chunk<T> w = load_chunk<kVec>(weight + c, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = v[k][j] * r * chunk_get(w, j);
      }
      if constexpr (kE4M3) {
        store_e4m3<kVec>(q + base + c, v[k], inv, n);
      } else {
        store_chunk<kVec>(out + base + c, v[k], n);
      }
    }
  }
}

// ------------------------------------------------------------------ its backward
// g = dout * w, xh = h * rstd, c = mean(g * xh): dres = dh + rstd * (g - xh * c), dx = dropout(dres), dw = sum(dout * xh).
// h is the stored one: in a 2-byte type dw and xh carry its half step.  (Forming h again from x and residual would read one
// more tensor, ten instead of nine tensor passes a step.)
//
// Bound by HBM.  Rows are owned as in the forward; a persistent grid keeps each thread on the same columns, so dw is summed
// in registers and leaves as one partial row a block, which fold_rows_kernel adds in a fixed order.
template <typename T, bool kVec, int kGroup, int kChunks>
__global__ void __launch_bounds__(kGroup < 256 ? 256 : kGroup)
norm_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ dh, const T* __restrict__ h, const float* __restrict__ rstd,
                const T* __restrict__ weight, Dropout d, T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partial,
                long long rows, int cols) {
  __shared__ float red[2 * 32];
  __shared__ float fold[kGroup == 32 ? 32 * kChunks * 8 : 1];
  const Mask mask(d);
  const bool drop = d.rng != nullptr;
  const int blocks = (cols + 3) / 4;
  const int lane = kGroup == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int per_block = kGroup == 32 ? blockDim.x / 32 : 1;
  float acc[kChunks][8];
#pragma unroll
  for (int k = 0; k < kChunks; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  for (long long row = static_cast<long long>(blockIdx.x) * per_block + (kGroup == 32 ? threadIdx.x / 32 : 0); row < rows;
       row += static_cast<long long>(gridDim.x) * per_block) {
    const long long base = row * cols;
    const float r = rstd[row];
    Chunk<T> o[kChunks], hh[kChunks], e[kChunks];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
      o[k] = load_chunk<kVec>(dout + base + c, n);
      hh[k] = load_chunk<kVec>(h + base + c, n);
      if (dh != nullptr) e[k] = load_chunk<kVec>(dh + base + c, n);
    }
    float dot = 0.f, unused = 0.f;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
      const Chunk<T> w = load_chunk<kVec>(weight + c, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = chunk_get(o[k], j) * (chunk_get(hh[k], j) * r);
        acc[k][j] += t;
        dot = fmaf(t, chunk_get(w, j), dot);
      }
    }
    row_reduce<kGroup, false>(dot, unused, red);
    const float m = dot / static_cast<float>(cols);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup), n = cols - c;
      const Chunk<T> w = load_chunk<kVec>(weight + c, n);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = r * (chunk_get(o[k], j) * chunk_get(w, j) - chunk_get(hh[k], j) * r * m);
        if (dh != nullptr) v[j] += chunk_get(e[k], j);
      }
      if (dres != nullptr) store_chunk<kVec>(dres + base + c, v, n);
      if (dx != nullptr) {
        if (drop && n > 0) mask.apply(v, static_cast<unsigned long long>(row) * blocks + c / 4);
        store_chunk<kVec>(dx + base + c, v, n);
      }
    }
  }
  if (partial == nullptr) return;
  float* mine = partial + static_cast<long long>(blockIdx.x) * cols;
  if constexpr (kGroup == 32) {
    // the warps of a block add up in turn
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) {
      if (static_cast<int>(threadIdx.x) / 32 == w) {
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float* f = fold + (k * 32 + lane) * 8 + j;
            *f = w == 0 ? acc[k][j] : *f + acc[k][j];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += blockDim.x) mine[c] = fold[c];
  } else {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = 8 * (lane + k * kGroup);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < cols) mine[c + j] = acc[k][j];
    }
  }
}

// ------------------------------------------------------------------ rows longer than registers hold
// The same mathematics for rows of more than kMaxCols columns: one block a row, which reads its operands twice (the second
// time mostly from L2) and keeps its dw sums in the partial row itself.
constexpr int kMaxCols = 16384, kColsLimit = 1 << 30;
constexpr int kLongThreads = 1024;
template <typename T, bool kVec, bool kE4M3>
__global__ void __launch_bounds__(kLongThreads)
norm_fwd_long_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ weight, float eps, Dropout d,
                     long long* __restrict__ used, T* __restrict__ h, T* __restrict__ out, float* __restrict__ rstd,
                     __nv_fp8_e4m3* __restrict__ q, float* __restrict__ scale, long long rows, int cols) {
  __shared__ float red[2 * 32];
  const Mask mask(d);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
  const int blocks = (cols + 3) / 4;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long long base = row * cols;
    auto value = [&](int c, float* v) {  // h of the chunk at c, unrounded
      const Chunk<T> a = load_chunk<kVec>(x + base + c, cols - c);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = chunk_get(a, j);
      if (d.rng != nullptr) mask.apply(v, static_cast<unsigned long long>(row) * blocks + c / 4);
      if (residual != nullptr) {
        const Chunk<T> b = load_chunk<kVec>(residual + base + c, cols - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += chunk_get(b, j);
      }
    };
    float sq = 0.f, top = 0.f, v[8];
    for (int c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads) {
      value(c, v);
      if (h != nullptr) store_chunk<kVec>(h + base + c, v, cols - c);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[j], v[j], sq);
      if (kE4M3) {
        Chunk<T> w;
        if (weight != nullptr) w = load_chunk<kVec>(weight + c, cols - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(weight != nullptr ? v[j] * chunk_get(w, j) : v[j]));
      }
    }
    row_reduce<kLongThreads, kE4M3>(sq, top, red);
    const float r = weight != nullptr ? rsqrtf(sq / static_cast<float>(cols) + eps) : 1.0f;
    float s = 1.0f;
    if (kE4M3) s = max_nan(top * r / 448.0f, 1.17549435e-38f);
    const float inv = 1.0f / s;
    if (threadIdx.x == 0) {
      if (kE4M3) scale[row] = s;
      else rstd[row] = r;
    }
    for (int c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads) {
      value(c, v);
      if (weight != nullptr) {
        const Chunk<T> w = load_chunk<kVec>(weight + c, cols - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * chunk_get(w, j);
      }
      if constexpr (kE4M3) store_e4m3<kVec>(q + base + c, v, inv, cols - c);
      else store_chunk<kVec>(out + base + c, v, cols - c);
    }
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kLongThreads)
norm_bwd_long_kernel(const T* __restrict__ dout, const T* __restrict__ dh, const T* __restrict__ h, const float* __restrict__ rstd,
                     const T* __restrict__ weight, Dropout d, T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partial,
                     long long rows, int cols) {
  __shared__ float red[2 * 32];
  const Mask mask(d);
  const int blocks = (cols + 3) / 4;
  float* mine = partial != nullptr ? partial + static_cast<long long>(blockIdx.x) * cols : nullptr;
  bool first = true;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, first = false) {
    const long long base = row * cols;
    const float r = rstd[row];
    float dot = 0.f, unused = 0.f;
    for (int c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads) {
      const int n = cols - c;
      const Chunk<T> o = load_chunk<kVec>(dout + base + c, n), hh = load_chunk<kVec>(h + base + c, n), w = load_chunk<kVec>(weight + c, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = chunk_get(o, j) * (chunk_get(hh, j) * r);
        dot = fmaf(t, chunk_get(w, j), dot);
        if (mine != nullptr && j < n) mine[c + j] = first ? t : mine[c + j] + t;
      }
    }
    row_reduce<kLongThreads, false>(dot, unused, red);
    const float m = dot / static_cast<float>(cols);
    for (int c = 8 * threadIdx.x; c < cols; c += 8 * kLongThreads) {
      const int n = cols - c;
      const Chunk<T> o = load_chunk<kVec>(dout + base + c, n), hh = load_chunk<kVec>(h + base + c, n), w = load_chunk<kVec>(weight + c, n);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r * (chunk_get(o, j) * chunk_get(w, j) - chunk_get(hh, j) * r * m);
      if (dh != nullptr) {
        const Chunk<T> e = load_chunk<kVec>(dh + base + c, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += chunk_get(e, j);
      }
      if (dres != nullptr) store_chunk<kVec>(dres + base + c, v, n);
      if (dx != nullptr) {
        if (d.rng != nullptr) mask.apply(v, static_cast<unsigned long long>(row) * blocks + c / 4);
        store_chunk<kVec>(dx + base + c, v, n);
      }
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
  if (rows < 0 || cols <= 0) return fail(kBadArgument, "rows must not be negative and cols must be positive");
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

// Threads of a row and chunks a thread, by the row's length: a warp to 1024 columns, then blocks of two chunks a thread
// (most bytes in flight for the registers), to 16384 columns.
struct RowShape {
  int group, chunks;
};
inline RowShape row_shape(int64_t cols) {
  const int64_t n = (cols + 7) / 8;
  if (n <= 32) return {32, 1};
  if (n <= 128) return {32, 4};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {512, 2};
  return {1024, 2};  // the long kernels take over beyond kMaxCols
}

inline int64_t row_blocks(int64_t rows, int64_t cols) {
  const RowShape s = row_shape(cols);
  const int64_t per_block = s.group == 32 ? 8 : 1, need = (rows + per_block - 1) / per_block;
  const int64_t cap = static_cast<int64_t>(sm_count()) * (2048 / (s.group < 256 ? 256 : s.group)) / 2;
  return need < cap ? need : cap;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class F>
int by_dtype(int dtype, F&& f) {
  if (dtype == 0) return f(__nv_bfloat16());
  if (dtype == 1) return f(__half());
  return f(float());
}
template <int kGroup, int kChunks>
struct Shape {
  [[maybe_unused]] static constexpr int group = kGroup;
  static constexpr int chunks = kChunks, threads = kGroup < 256 ? 256 : kGroup;
};
// chunks = 0: the kernel for long rows
template <class F>
int by_shape(int64_t cols, F&& f) {
  const RowShape s = row_shape(cols);
  if (cols > kMaxCols) return f(Shape<kLongThreads, 0>());
  if (s.group == 32) return s.chunks == 1 ? f(Shape<32, 1>()) : f(Shape<32, 4>());
  if (s.group == 256) return f(Shape<256, 2>());
  if (s.group == 512) return f(Shape<512, 2>());
  return f(Shape<1024, 2>());
}
template <class F>
int by_vec(bool vec, F&& f) {
  return vec ? f(std::true_type()) : f(std::false_type());
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
  if (cols % 4 == 0) {
    cols *= rows;
    rows = 1;
  }
  const long long need = (rows * ((cols + 7) / 8) + kDropThreads * kDropUnroll - 1) / (kDropThreads * kDropUnroll);
  const long long cap = static_cast<long long>(sm_count()) * 8;
  const int grid = static_cast<int>(need < cap ? need : cap);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_vec(rows == 1 && cols % 8 == 0 && aligned16(x) && aligned16(out), [&](auto vec) {
      dropout_kernel<T, decltype(vec)::value><<<grid, kDropThreads, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(x), static_cast<T*>(out), rows, cols, d, reinterpret_cast<long long*>(rng_used));
      return launch_check("dropout launch");
    });
  });
}

extern "C" int coda_b200_add_rmsnorm_fwd(const void* x, const void* residual, const void* weight, float eps, double p, const int64_t* rng,
                                         int64_t stream_id, int64_t* rng_used, void* h, void* out, float* rstd, int64_t rows,
                                         int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc == kOk && cols > kColsLimit) rc = fail(kBadArgument, "cols must not exceed 2^30");
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !weight || !out || !rstd) return fail(kBadArgument, "NULL pointer");
  const int grid = static_cast<int>(row_blocks(rows, cols));
  const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(h) && aligned16(out);
  return by_dtype(dtype, [&](auto t) {
    return by_shape(cols, [&](auto shape) {
      return by_vec(vec, [&](auto v) {
        using T = decltype(t);
        using S = decltype(shape);
        auto kern = [] {
          if constexpr (S::chunks == 0) return norm_fwd_long_kernel<T, decltype(v)::value, false>;
          else return norm_fwd_kernel<T, decltype(v)::value, S::group, S::chunks, false>;
        }();
        kern<<<grid, S::threads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), eps, d,
            reinterpret_cast<long long*>(rng_used), static_cast<T*>(h), static_cast<T*>(out), rstd, nullptr, nullptr, rows,
            static_cast<int>(cols));
        return launch_check("add_rmsnorm forward launch");
      });
    });
  });
}

extern "C" int coda_b200_rows_e4m3(const void* x, const void* residual, const void* weight, float eps, void* h, void* q, float* scale,
                                   int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc == kOk && cols > kColsLimit) rc = fail(kBadArgument, "cols must not exceed 2^30");
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !q || !scale) return fail(kBadArgument, "NULL pointer");
  const Dropout d{nullptr, 0u, 0u, 1.0f};
  const int grid = static_cast<int>(row_blocks(rows, cols));
  const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(h) &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  return by_dtype(dtype, [&](auto t) {
    return by_shape(cols, [&](auto shape) {
      return by_vec(vec, [&](auto v) {
        using T = decltype(t);
        using S = decltype(shape);
        auto kern = [] {
          if constexpr (S::chunks == 0) return norm_fwd_long_kernel<T, decltype(v)::value, true>;
          else return norm_fwd_kernel<T, decltype(v)::value, S::group, S::chunks, true>;
        }();
        kern<<<grid, S::threads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), eps, d, nullptr, static_cast<T*>(h),
            nullptr, nullptr, static_cast<__nv_fp8_e4m3*>(q), scale, rows, static_cast<int>(cols));
        return launch_check("e4m3 rows launch");
      });
    });
  });
}

extern "C" int64_t coda_b200_add_rmsnorm_bwd_scratch_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : row_blocks(rows, cols) * cols * static_cast<int64_t>(sizeof(float));
}

extern "C" int coda_b200_add_rmsnorm_bwd(const void* dout, const void* dh, const void* h, const float* rstd, const void* weight, double p,
                                         const int64_t* rng, int64_t stream_id, void* dx, void* dres, void* dweight, void* scratch,
                                         int64_t scratch_bytes, int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_extents(rows, cols, dtype);
  if (rc == kOk && cols > kColsLimit) rc = fail(kBadArgument, "cols must not exceed 2^30");
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!dout || !h || !rstd || !weight) return fail(kBadArgument, "NULL pointer");
  if (dweight != nullptr && (scratch == nullptr || scratch_bytes < coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols)))
    return fail(kBadArgument, "the weight gradient needs coda_b200_add_rmsnorm_bwd_scratch_bytes of scratch");
  const int blocks = static_cast<int>(row_blocks(rows, cols)), n = static_cast<int>(cols);
  const bool vec = cols % 8 == 0 && aligned16(dout) && aligned16(dh) && aligned16(h) && aligned16(weight) && aligned16(dx) && aligned16(dres);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int rc2 = by_shape(cols, [&](auto shape) {
      return by_vec(vec, [&](auto v) {
        using S = decltype(shape);
        auto kern = [] {
          if constexpr (S::chunks == 0) return norm_bwd_long_kernel<T, decltype(v)::value>;
          else return norm_bwd_kernel<T, decltype(v)::value, S::group, S::chunks>;
        }();
        kern<<<blocks, S::threads, 0, st>>>(
            static_cast<const T*>(dout), static_cast<const T*>(dh), static_cast<const T*>(h), rstd, static_cast<const T*>(weight), d,
            static_cast<T*>(dx), static_cast<T*>(dres), dweight != nullptr ? static_cast<float*>(scratch) : nullptr, rows, n);
        return launch_check("add_rmsnorm backward launch");
      });
    });
    if (rc2 != kOk || dweight == nullptr) return rc2;
    fold_rows_kernel<T><<<(n + 31) / 32, 1024, 0, st>>>(static_cast<const float*>(scratch), blocks, n, static_cast<T*>(dweight));
    return launch_check("add_rmsnorm weight gradient launch");
  });
}
