// Row kernels around the fused linears: counter-based dropout, the residual addition with dropout and RMS norm
// (forward and backward), and rows leaving as e4m3 values with one scale each.  Matrices are dense [rows, cols] of
// bf16, fp16 or fp32; all arithmetic is fp32.  See include/coda_b200.h for the contract.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "../../include/coda_b200.h"
#include "gemm_host.cuh"

using namespace cb;

namespace {

// ------------------------------------------------------------------ chunks
// A thread works on chunks of 8 consecutive elements, held as loaded (2-byte types: 4 registers, fp32: 8).  A chunk always
// starts at a multiple of 8 elements of the whole (dense, 16-byte aligned) matrix, so it moves in 16-byte accesses whatever
// the row's length.  With cols % 8 != 0 (kShift) a row therefore begins `off` = row * cols mod 8 elements into its first
// chunk; elements of a chunk that belong to the neighbouring rows are read, masked to zero before use, and never written.
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

// The elements of a chunk that a thread may touch: [lo, hi).  Without kShift a chunk is whole or not there at all.
template <bool kShift>
struct Span {
  int c0;  // column of element 0 (kShift: may be negative)
  int lo, hi;
  __device__ Span(int first, int cols) : c0(first), lo(first < 0 ? -first : 0), hi(cols - first < 8 ? cols - first : 8) {}
  __device__ bool any() const { return kShift ? hi > lo : hi > 0; }
  __device__ bool whole() const { return kShift ? (lo == 0 && hi == 8) : hi > 0; }
};

template <typename T>
__device__ __forceinline__ Chunk<T> load_whole(const T* p) {
  Chunk<T> c;
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) {
    const uint4 u = *(reinterpret_cast<const uint4*>(p) + k);
    c.w[4 * k] = u.x;
    c.w[4 * k + 1] = u.y;
    c.w[4 * k + 2] = u.z;
    c.w[4 * k + 3] = u.w;
  }
  return c;
}
template <typename T>
__device__ __forceinline__ Chunk<T> zero_chunk() {
  Chunk<T> c;
#pragma unroll
  for (int k = 0; k < static_cast<int>(2 * sizeof(T)); ++k) c.w[k] = 0u;
  return c;
}
// elements [lo, hi) one by one, zero elsewhere
template <typename T>
__device__ __forceinline__ Chunk<T> load_some(const T* p, int lo, int hi) {
  Chunk<T> c = zero_chunk<T>();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j >= lo && j < hi) {
      if constexpr (sizeof(T) == 4) c.w[j] = __float_as_uint(p[j]);
      else c.w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[j]) << (16 * (j & 1));
    }
  return c;
}
// The chunk at p as it is, neighbours' elements included; `left` = elements from p to the end of the matrix (a chunk that
// reaches beyond it is read one by one).  mask_chunk takes the neighbours out, where the values are used: a load that is
// masked at once is waited for at once, row by row in the warps at a row's ends (backward 16384 x 4095: 383 us that way, 223 us
// so).
template <bool kShift, typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p, const Span<kShift>& s, long long left) {
  if (!s.any()) return zero_chunk<T>();
  if constexpr (kShift) {
    if (left < 8) return load_some(p, 0, static_cast<int>(left));
  }
  return load_whole(p);
}
template <bool kShift, typename T>
__device__ __forceinline__ void mask_chunk(Chunk<T>& c, const Span<kShift>& s) {
  if constexpr (kShift) {
    if (s.whole()) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < s.lo || j >= s.hi) {
        if constexpr (sizeof(T) == 4) c.w[j] = 0u;
        else c.w[j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
      }
  }
}
template <bool kShift, typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* v, const Span<kShift>& s) {
  if (s.whole()) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
  } else if constexpr (kShift) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= s.lo && j < s.hi) p[j] = from_f32<T>(v[j]);
  }
}

// ------------------------------------------------------------------ the bits of h below its 2-byte type
// h is stored in T, half a step off; what is summed over rows of it (the weight gradient) would carry that rounding beside its
// own, 1.4 times the error.  So the forward also leaves four bits an element.  With v the fp32 value and hi = v rounded to T, the
// difference of their bit patterns (sign and magnitude, so it is monotone across binades) lies within the half step kHalf; n =
// floor((hi - v + kHalf) 15 / (2 kHalf)) is 0 .. 15, 7 where they are equal, and hi + (7 - n) kUnit gives v back to half a unit:
// 2^-11 of its size (bf16; fp16 2^-14, for normal numbers), a fifteenth of the half step, which does not show in a sum's error
// (16384 x 4096, against 64 bits: bf16 2.3e-3 without these bits, 1.7e-3 with them, which is the rounding of the sum).
// n is the top nibble of a product with a power of two times 15, and is shifted from there into the chunk's word, the first element's
// into the top.
// The words follow the chunks, and where two rows may share a chunk its place moves on by one a row, so that no word belongs to two.
template <typename T>
struct Low;
template <>
struct Low<__nv_bfloat16> {
  static constexpr int kHalf = 1 << 15, kUnit = 4369;
};
template <>
struct Low<__half> {
  static constexpr int kHalf = 1 << 12, kUnit = 546;
};
constexpr long long low_words(long long rows, long long cols) { return cols % 8 == 0 ? rows * (cols / 8) : (rows * cols + 7) / 8 + rows; }
// the word of the chunk of `row` that begins at element e of the matrix
template <bool kShift>
__device__ __forceinline__ long long low_at(long long e, long long row) {
  return (e >> 3) + (kShift ? row : 0);
}

template <typename T>
__device__ __forceinline__ uint32_t low_word(const float* v) {
  Chunk<T> c;
#pragma unroll
  for (int j = 0; j < 4; ++j) c.w[j] = pack2(v[2 * j], v[2 * j + 1], T());
  uint32_t word = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int u = __float_as_int(chunk_get(c, j)) - __float_as_int(v[j]) + Low<T>::kHalf;
    // below its normal numbers and above its largest fp16 is further off
    if constexpr (std::is_same<T, __half>::value) u = min(max(u, 0), 2 * Low<T>::kHalf);
    word = __funnelshift_l(static_cast<uint32_t>(u) * (0x78000000u / Low<T>::kHalf), word, 4);
  }
  return word;
}
// The nibbles of a word as bytes: of the odd elements and of the even ones, the last pair's first.
struct LowBytes {
  uint32_t odd, even;
  __device__ __forceinline__ explicit LowBytes(uint32_t word) : odd(word & 0x0f0f0f0fu), even((word >> 4) & 0x0f0f0f0fu) {}
  __device__ __forceinline__ int get(int j) const { return static_cast<int>(__byte_perm(j & 1 ? odd : even, 0u, 0x4440 | (3 - (j >> 1)))); }
};
// element j of a chunk with the bits below its type (7 kUnit = 0x7777 fits the bits that bf16 leaves empty)
__device__ __forceinline__ float chunk_get_whole(const Chunk<__nv_bfloat16>& c, const LowBytes& low, int j) {
  const uint32_t top = j & 1 ? (c.w[j >> 1] & 0xffff0000u) | 0x7777u : __byte_perm(c.w[j >> 1], 0x7777u, 0x1054);
  return __int_as_float(static_cast<int>(top) - low.get(j) * Low<__nv_bfloat16>::kUnit);
}
__device__ __forceinline__ float chunk_get_whole(const Chunk<__half>& c, const LowBytes& low, int j) {
  return __int_as_float(__float_as_int(chunk_get(c, j)) + (7 - low.get(j)) * Low<__half>::kUnit);
}

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The scale of a row of e4m3 values, and what divides by it.  Both quotients have to be the correctly rounded ones: values of
// a 2-byte type lie exactly between two e4m3 values all the time (with max|y| = 21 / 8, say, where the scale is 3 / 512 and
// y / scale = 512 y / 3), and a scale or a quotient one step off moves them all to the same side (fp32's 1 / 448 is too large:
// a product with it is one step off in every other row whose maximum is a multiple of 7).  A division for every element made the
// kernel slower than its memory traffic, though.  So: with inv = 1 / s rounded correctly and q = v inv, the residual v - q s
// is exact in an fma, and q + residual * inv is v / s rounded correctly (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990; quantize 16384 x 4096 bf16: 44 us, 41 us with q alone).  Where the residual falls
// below the smallest fp32, |v| < 2^-100, the last bit may be lost.
struct RowScale {
  float scale, inv, s;  // s: the scale, or 0 if that is infinite, so that finite values over it come out as 0
  __device__ explicit RowScale(float top)
      : scale(max_nan(top / 448.0f, 1.17549435e-38f)), inv(1.0f / scale), s(isinf(scale) ? 0.0f : scale) {}
  __device__ float over(float v) const {
    const float q = v * inv;
    return fmaf(fmaf(-q, s, v), inv, q);
  }
};

// Values over their row's scale as e4m3, rounded once more; saturation keeps 448 (1 + 2^-23) at 448.
template <bool kShift>
__device__ __forceinline__ void store_e4m3(__nv_fp8_e4m3* p, const float* v, const RowScale& by, const Span<kShift>& s) {
  uint32_t e[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) e[j] = __nv_cvt_float2_to_fp8x2(make_float2(by.over(v[2 * j]), by.over(v[2 * j + 1])), __NV_SATFINITE, __NV_E4M3);
  if (s.whole()) {
    *reinterpret_cast<uint2*>(p) = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
  } else if constexpr (kShift) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= s.lo && j < s.hi) p[j].__x = static_cast<__nv_fp8_storage_t>(e[j / 2] >> (8 * (j & 1)));
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

// Both halves of a 32 x 32-bit product.  Written out as one instruction (kAsm) it makes the dropout kernel, four blocks at
// once, 8 % faster; in the norm kernels, two at once, it cost registers (backward 16384 x 4096 bf16 142 instead of 123 us).
template <bool kAsm>
__device__ __forceinline__ void mul_wide(uint32_t a, uint32_t b, uint32_t& hi, uint32_t& lo) {
  if constexpr (!kAsm) {
    const unsigned long long t = static_cast<unsigned long long>(a) * b;
    hi = static_cast<uint32_t>(t >> 32);
    lo = static_cast<uint32_t>(t);
    return;
  }
  asm("{\n\t.reg .b64 t;\n\tmul.wide.u32 t, %2, %3;\n\tmov.b64 {%1, %0}, t;\n\t}" : "=r"(hi), "=r"(lo) : "r"(a), "r"(b));
}

struct Mask {
  uint32_t k0, k1, lo, first, second;  // seed; round 1 of the words that do not depend on the block (see words)
  uint32_t threshold;
  float scale;

  __device__ explicit Mask(const Dropout& d) : threshold(d.threshold), scale(d.scale) {
    const unsigned long long seed = static_cast<unsigned long long>(__ldg(d.rng));
    k0 = static_cast<uint32_t>(seed);
    k1 = static_cast<uint32_t>(seed >> 32);
    uint32_t hi;
    mul_wide<false>(static_cast<uint32_t>(__ldg(d.rng + 1)), 0xCD9E8D57u, hi, lo);
    first = hi ^ k0;
    second = d.stream ^ k1;
  }
  // The words of kN blocks, in step: the key words advance once for all of them, which costs fewer instructions than a key
  // schedule each and fewer registers than one that is kept (16384 x 4095 bf16: 137 us with it kept, 118 us so).
  template <int kN>
  __device__ __forceinline__ void words(const unsigned long long (&block)[kN], uint32_t* u) const {
    uint32_t c0[kN], c1[kN], c2[kN], c3[kN], a = k0, b = k1;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      uint32_t hi0;
      mul_wide<(kN > 3)>(static_cast<uint32_t>(block[n]), 0xD2511F53u, hi0, c3[n]);
      c0[n] = first ^ static_cast<uint32_t>(block[n] >> 32);
      c1[n] = lo;
      c2[n] = hi0 ^ second;
    }
#pragma unroll
    for (int i = 1; i < 10; ++i) {
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        uint32_t hi0, lo0, hi1, lo1;
        mul_wide<(kN > 3)>(c0[n], 0xD2511F53u, hi0, lo0);
        mul_wide<(kN > 3)>(c2[n], 0xCD9E8D57u, hi1, lo1);
        c0[n] = hi1 ^ c1[n] ^ a;
        c1[n] = lo1;
        c2[n] = hi0 ^ c3[n] ^ b;
        c3[n] = lo0;
      }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      u[4 * n] = c0[n];
      u[4 * n + 1] = c1[n];
      u[4 * n + 2] = c2[n];
      u[4 * n + 3] = c3[n];
    }
  }
  // the words of 8 elements that begin at word `phase` (0 .. 3) of `block`
  template <bool kShift>
  __device__ __forceinline__ void words8(unsigned long long block, int phase, uint32_t* u) const {
    if constexpr (kShift) {
      if (phase != 0) {
        words<3>({block, block + 1, block + 2}, u);
        if (phase & 1) {
#pragma unroll
          for (int j = 0; j < 11; ++j) u[j] = u[j + 1];
        }
        if (phase & 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = u[j + 2];
        }
        return;
      }
    }
    words<2>({block, block + 1}, u);
  }
  // a dropped value is +0 whatever it held
  __device__ __forceinline__ float apply(float v, uint32_t u) const { return u >= threshold ? v * scale : 0.0f; }
  struct Words {
    uint32_t u[12];
  };
  // the words of the 8 values of `row` from column c0 on (kShift: c0 may be any, also below zero, where they are not used)
  template <bool kShift>
  __device__ __forceinline__ Words words_at(long long row, int blocks, int c0) const {
    Words w;
    words8<kShift>(static_cast<unsigned long long>(row * blocks + (c0 >> 2)), kShift ? c0 & 3 : 0, w.u);
    return w;
  }
  __device__ __forceinline__ void apply8(float* v, const Words& w) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = apply(v[j], w.u[j]);
  }
};
struct NoMask {
  struct Words {};
  __device__ explicit NoMask(const Dropout&) {}
  template <bool kShift>
  __device__ __forceinline__ Words words_at(long long, int, int) const {
    return {};
  }
  __device__ __forceinline__ void apply8(float*, const Words&) const {}
};
template <bool kDrop>
using MaskOf = typename std::conditional<kDrop, Mask, NoMask>::type;

// The [seed, step] a forward used, for its backward.
__device__ __forceinline__ void note_used(const Dropout& d, long long* used) {
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x < 2) used[threadIdx.x] = d.rng != nullptr ? d.rng[threadIdx.x] : 0;
}

// (sum of a, max of b >= 0) over the threads of a row: kLanes neighbouring lanes of a warp, or (0) the whole block of at
// most 32 warps.  `red` is two buffers of 64 floats used in turn, `turn` counts the calls: a buffer is written again only
// after the synchronisation of the call in between, so one is enough.
template <int kLanes, bool kMax>
__device__ __forceinline__ void row_reduce(float& a, float& b, float* red, int& turn) {
  // the lanes of a row run together; those of the warp's other rows may have left the loop
  constexpr uint32_t kOnes = kLanes == 0 || kLanes == 32 ? 0xffffffffu : (1u << (kLanes & 31)) - 1u;
  const uint32_t lanes = kLanes == 0 || kLanes == 32 ? kOnes : kOnes << (threadIdx.x & 31 & ~(kLanes - 1));
#pragma unroll
  for (int o = kLanes == 0 ? 16 : kLanes / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(lanes, a, o);
    if (kMax) b = max_nan(b, __shfl_xor_sync(lanes, b, o));
  }
  if constexpr (kLanes == 0) {
    float* r = red + 64 * (turn++ & 1);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
      r[threadIdx.x >> 5] = a;
      if (kMax) r[32 + (threadIdx.x >> 5)] = b;
    }
    __syncthreads();
    a = lane < warps ? r[lane] : 0.f;
    if (kMax) b = lane < warps ? r[32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (kMax) b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
  }
}

// ------------------------------------------------------------------ dropout alone
// A stream of chunks of the whole matrix, drop_unroll() of them in flight a thread, by four blocks an SM (eight: 158 instead of
// 147 us for 16384 x 14336 bf16 without a mask; 32 bytes a thread suffice, a second fp32 chunk costs 52 instead of 43 us at 8192
// x 4096).  Without the mask, and in fp32, bound by HBM (6.2 to 6.4 TB/s).  With it a 2-byte type is bound by the integer
// multiplier, 19 wide products for 4 elements: 225 us, one element a nanosecond, whatever the occupancy.
constexpr int kDropThreads = 256, kDropBlocksPerSm = 4;
constexpr int drop_unroll(int elem_bytes) { return elem_bytes == 4 ? 1 : 2; }
template <typename T, bool kShift, bool kDrop>
__global__ void __launch_bounds__(kDropThreads, kDropBlocksPerSm)
dropout_kernel(const T* __restrict__ x, T* __restrict__ out, long long total, long long cols, Dropout d, long long* __restrict__ used) {
  constexpr int kUnroll = drop_unroll(sizeof(T));
  const MaskOf<kDrop> mask(d);
  note_used(d, used);
  const long long chunks = (total + 7) / 8, blocks = (cols + 3) / 4;
  const long long stride = static_cast<long long>(gridDim.x) * kDropThreads;
  for (long long i0 = blockIdx.x * static_cast<long long>(kDropThreads) + threadIdx.x; i0 < chunks; i0 += stride * kUnroll) {
    Chunk<T> in[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const long long e = 8 * (i0 + k * stride);
      if (e + 8 <= total) in[k] = load_whole(x + e);
      else in[k] = load_some(x + e, 0, e < total ? static_cast<int>(total - e) : 0);
    }
    uint32_t all[kUnroll * 8];
    if constexpr (kDrop && !kShift) {  // cols % 4 == 0: a row's blocks follow the previous row's
      unsigned long long block[2 * kUnroll];
#pragma unroll
      for (int k = 0; k < 2 * kUnroll; ++k) block[k] = 2 * static_cast<unsigned long long>(i0 + k / 2 * stride) + (k & 1);
      mask.template words<2 * kUnroll>(block, all);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const long long e = 8 * (i0 + k * stride);
      if (e >= total) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = chunk_get(in[k], j);
      if constexpr (kDrop) {
        uint32_t u[12];
        if constexpr (!kShift) {
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = all[8 * k + j];
        } else {
          long long row = total <= 0xffffffffLL ? static_cast<uint32_t>(e) / static_cast<uint32_t>(cols) : e / cols;
          long long c = e - row * cols;
          mask.template words8<true>(static_cast<unsigned long long>(row * blocks + c / 4), static_cast<int>(c & 3), u);
          if (c + 8 > cols) {  // the next row (or rows) begins inside the chunk
            uint32_t t[4] = {0u, 0u, 0u, 0u};
            bool next = false;
#pragma unroll
            for (int j = 0; j < 8; ++j, ++c) {
              if (c == cols) {
                c = 0;
                ++row;
                next = true;
              }
              if (next) {
                const int q = static_cast<int>(c & 3);
                if (q == 0) mask.template words<1>({static_cast<unsigned long long>(row * blocks + c / 4)}, t);
                u[j] = q == 0 ? t[0] : q == 1 ? t[1] : q == 2 ? t[2] : t[3];
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = mask.apply(v[j], u[j]);
      }
      const long long left = total - e;
      store_chunk<true>(out + e, v, Span<true>(0, left < 8 ? static_cast<int>(left) : 8));
    }
  }
}

// ------------------------------------------------------------------ residual + dropout(x), RMS norm
// h = residual + dropout(x) (x alone without a residual); rstd = rsqrt(mean(h^2) + eps), taken of the unrounded h; out =
// h * rstd * w.  kE4M3: out leaves as e4m3 values q with scale = max(max|out| / 448, 2^-126), q = out / scale rounded
// to e4m3; without a weight the rows are converted as they are.
//
// Bound by HBM: every tensor is read or written once.  The block (or kLanes lanes of a warp) owns a row and keeps its h in
// registers, kChunks chunks a thread; the grid is what fits the SMs at once, and a row's successor is loaded while the row is reduced
// and written.  A thread stays on the same columns for all of its rows (kShift: the grid's row stride is a multiple of 8, so
// `off` stays too), so the weights are loaded once.
constexpr int kWarpBlock = 256, kMaxThreads = 512;
// Registers a thread, and so threads an SM.  Forward: two chunks of a 2-byte type fit 64, of fp32 80; four chunks take 128.
// Backward: with sums and the next row's loads two chunks of a 2-byte type take 128 (16384 x 4096 bf16: 96 us; 102 us with 80
// registers and no loads ahead, 133 us with 96 registers and loads ahead); fp32, which loads nothing ahead, takes 96 (16384 x
// 4096: 203 us, 128: 236 us), but 128 with dropout (8192 x 8192: 220 us, 96: 255 us).  With the shift 96 (16384 x 4095 bf16, forward,
// backward, e4m3: 96, 155 and 107 us; with 80 105, 191 and 121 us), but 80 for one chunk a thread (300000 x 129: 98 and 133 us;
// with 96 114 and 164 us) and for fp32 forward (16384 x 2047: 89 us, 96: 105 us).
constexpr int fwd_regs(int elem_bytes, bool shift, int chunks, bool e4m3) {
  if (chunks == 4) return 128;
  if (shift) return chunks == 1 || (elem_bytes == 4 && !e4m3) ? 80 : 96;
  return elem_bytes == 4 ? 80 : 64;
}
constexpr int bwd_regs(int elem_bytes, bool shift, bool drop, int chunks) {
  if (shift) return chunks == 1 ? 80 : 96;
  return elem_bytes == 4 && !drop ? 96 : 128;
}
constexpr int threads_per_sm(int regs) { return 512 / regs * 4 * 32; }  // whole warps in each quarter of the SM

template <int kLanes>
struct RowLoop {
  static constexpr int kPerBlock = kLanes == 0 ? 1 : kWarpBlock / (kLanes == 0 ? 1 : kLanes);  // rows of a block
  long long row, step;
  int tid, width;  // this thread and the number of threads of the row
  __device__ RowLoop()
      : row(kLanes == 0 ? blockIdx.x : static_cast<long long>(blockIdx.x) * kPerBlock + threadIdx.x / (kLanes == 0 ? 1 : kLanes)),
        step(static_cast<long long>(gridDim.x) * kPerBlock),
        tid(kLanes == 0 ? threadIdx.x : threadIdx.x & (kLanes - 1)),
        width(kLanes == 0 ? blockDim.x : kLanes) {}
  // elements of the row's first chunk that belong to the row before it (kShift)
  __device__ int offset(int cols) const { return static_cast<int>((row * cols) & 7); }
};

template <typename T, bool kShift, bool kDrop, int kLanes, int kChunks, bool kE4M3>
__global__ void __maxnreg__(fwd_regs(sizeof(T), kShift, kChunks, kE4M3))
norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ weight, float eps, Dropout d,
                long long* __restrict__ used, T* __restrict__ h, uint32_t* __restrict__ low, T* __restrict__ out, float* __restrict__ rstd,
                __nv_fp8_e4m3* __restrict__ q, float* __restrict__ scale, long long rows, int cols) {
  __shared__ float red[kLanes != 0 ? 1 : 128];
  int turn = 0;
  const MaskOf<kDrop> mask(d);
  note_used(d, used);
  const int blocks = (cols + 3) / 4;
  const long long total = rows * cols;
  RowLoop<kLanes> at;
  if (at.row >= rows) return;  // all threads of the row leave together
  const int off = kShift ? at.offset(cols) : 0;
  auto span = [&](int k) { return Span<kShift>(8 * (at.tid + k * at.width) - off, cols); };
  Chunk<T> w[kChunks], a[kChunks], b[kChunks];
#pragma unroll
  for (int k = 0; k < kChunks; ++k)
    if (weight != nullptr) w[k] = kShift ? load_some(weight + span(k).c0, span(k).lo, span(k).hi) : load_chunk(weight + span(k).c0, span(k), 8);
  auto load = [&](long long row) {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const Span<kShift> s = span(k);
      const long long e = row * cols + s.c0;
      a[k] = load_chunk(x + e, s, total - e);
      if (residual != nullptr) b[k] = load_chunk(residual + e, s, total - e);
    }
  };
  load(at.row);
  for (; at.row < rows; at.row += at.step) {
    const long long base = at.row * cols;
    float v[kChunks][8], sq = 0.f, top = 0.f;
    // the mask first: it needs none of the row's values, which are still on their way (16384 x 4096 bf16: 98 us, 106 us with the
    // mask where it is used; 8192 x 8192 fp32 165 and 192 us)
    typename MaskOf<kDrop>::Words u[kChunks];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) u[k] = mask.template words_at<kShift>(at.row, blocks, span(k).c0);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const Span<kShift> s = span(k);
      mask_chunk(a[k], s);
      if (residual != nullptr) mask_chunk(b[k], s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = chunk_get(a[k], j);
      mask.apply8(v[k], u[k]);
      if (residual != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] += chunk_get(b[k], j);
      }
      // (elements outside the row are zero: they were masked, and dropout keeps zeros)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sq = fmaf(v[k][j], v[k][j], sq);
        if (kE4M3) top = max_nan(top, fabsf(weight != nullptr ? v[k][j] * chunk_get(w[k], j) : v[k][j]));
      }
    }
    if (at.row + at.step < rows) load(at.row + at.step);
    if (h != nullptr) {
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        store_chunk(h + base + span(k).c0, v[k], span(k));
        if constexpr (!kE4M3 && sizeof(T) == 2) {
          if (low != nullptr && span(k).any()) low[low_at<kShift>(base + span(k).c0, at.row)] = low_word<T>(v[k]);
        }
      }
    }
    row_reduce<kLanes, kE4M3>(sq, top, red, turn);
    const float r = weight != nullptr ? rsqrtf(sq / static_cast<float>(cols) + eps) : 1.0f;
    const RowScale by(top * r);
    if (at.tid == 0) {
      if (kE4M3) scale[at.row] = by.scale;
      else rstd[at.row] = r;
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const Span<kShift> s = span(k);
      if (weight != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = v[k][j] * r * chunk_get(w[k], j);
      }
      if constexpr (kE4M3) store_e4m3(q + base + s.c0, v[k], by, s);
      else store_chunk(out + base + s.c0, v[k], s);
    }
  }
}

// ------------------------------------------------------------------ its backward
// g = dout * w, xh = h * rstd, c = mean(g * xh): dres = dh + rstd * (g - xh * c), dx = dropout(dres), dw = sum(dout * xh).
// h is the stored one, with the bits below a 2-byte type where the forward has left them.  (Half a byte an element more each way:
// 16384 x 4096 bf16 198 us a step without them, 210 with; 231 and 250 with dropout.  The other times of residual norms in
// this file's comments were taken without them.  Forming h again from x and residual would read one tensor more, and the node
// would keep one more.)
//
// Bound by HBM, and laid out as the forward; dw is summed in registers over a thread's rows and leaves as one partial row a
// block, which fold_rows_kernel adds in a fixed order.
template <typename T, bool kShift, bool kDrop, bool kLow, int kLanes, int kChunks>
__global__ void __maxnreg__(bwd_regs(sizeof(T), kShift, kDrop, kChunks))
norm_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ dh, const T* __restrict__ h, const uint32_t* __restrict__ low,
                const float* __restrict__ rstd, const T* __restrict__ weight, Dropout d, T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partial,
                long long rows, int cols) {
  // the next row's loads need as many registers again
  constexpr bool kPrefetch = !kShift && sizeof(T) == 2;
  __shared__ float red[kLanes != 0 ? 1 : 128];
  __shared__ float fold[kLanes != 0 ? 256 : 1];
  int turn = 0;
  const MaskOf<kDrop> mask(d);
  const int blocks = (cols + 3) / 4;
  const long long total = rows * cols;
  RowLoop<kLanes> at;
  const int off = kShift ? at.offset(cols) : 0;
  auto span = [&](int k) { return Span<kShift>(8 * (at.tid + k * at.width) - off, cols); };
  struct Row {
    Chunk<T> o[kChunks], h[kChunks], e[kChunks];
    uint32_t low[kLow ? kChunks : 1];
    float r;
  };
  auto load = [&](long long row, Row& in) {
    in.r = rstd[row];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const Span<kShift> s = span(k);
      const long long e = row * cols + s.c0;
      in.o[k] = load_chunk(dout + e, s, total - e);
      in.h[k] = load_chunk(h + e, s, total - e);
      if constexpr (kLow) in.low[k] = s.any() ? low[low_at<kShift>(e, row)] : 0u;
      if (dh != nullptr) in.e[k] = load_chunk(dh + e, s, total - e);
    }
  };
  Chunk<T> w[kChunks];
  float acc[kChunks][8];
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    w[k] = kShift ? load_some(weight + span(k).c0, span(k).lo, span(k).hi) : load_chunk(weight + span(k).c0, span(k), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  }
  Row cur, nxt;
  if (kPrefetch && at.row < rows) load(at.row, cur);
  for (; at.row < rows; at.row += at.step) {
    if constexpr (kPrefetch) {
      if (at.row + at.step < rows) load(at.row + at.step, nxt);
    } else {
      load(at.row, cur);
    }
    const long long base = at.row * cols;
    const float r = cur.r;
    float dot = 0.f, unused = 0.f, xh[kChunks][8];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      mask_chunk(cur.o[k], span(k));
      mask_chunk(cur.h[k], span(k));
      const LowBytes bits(kLow ? cur.low[k] : 0u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (kLow) xh[k][j] = chunk_get_whole(cur.h[k], bits, j) * r;
        else xh[k][j] = chunk_get(cur.h[k], j) * r;
        const float t = chunk_get(cur.o[k], j) * xh[k][j];
        acc[k][j] += t;
        dot = fmaf(t, chunk_get(w[k], j), dot);
      }
    }
    row_reduce<kLanes, false>(dot, unused, red, turn);
    const float m = dot / static_cast<float>(cols);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const Span<kShift> s = span(k);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = r * (chunk_get(cur.o[k], j) * chunk_get(w[k], j) - xh[k][j] * m);
        if (dh != nullptr) v[j] += chunk_get(cur.e[k], j);
      }
      if (dres != nullptr) store_chunk(dres + base + s.c0, v, s);
      if (dx != nullptr) {
        // (the test costs 2-byte types 3 us at 16384 x 4096; without it the fp32 form spills: 8192 x 8192 300 instead of 218 us)
        if (sizeof(T) == 2 || s.any()) mask.apply8(v, mask.template words_at<kShift>(at.row, blocks, s.c0));
        store_chunk(dx + base + s.c0, v, s);
      }
    }
    if constexpr (kPrefetch) cur = nxt;
  }
  if (partial == nullptr) return;
  float* mine = partial + static_cast<long long>(blockIdx.x) * cols;
  if constexpr (kLanes != 0) {
    // the rows' lanes add up in turn
    for (int c = threadIdx.x; c < cols; c += kWarpBlock) fold[c] = 0.f;
    __syncthreads();
    for (int i = 0; i < RowLoop<kLanes>::kPerBlock; ++i) {
      if (static_cast<int>(threadIdx.x) / kLanes == i) {
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j >= span(k).lo && j < span(k).hi) fold[span(k).c0 + j] += acc[k][j];
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += kWarpBlock) mine[c] = fold[c];
  } else {
#pragma unroll
    for (int k = 0; k < kChunks; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= span(k).lo && j < span(k).hi) mine[span(k).c0 + j] = acc[k][j];
  }
}

// ------------------------------------------------------------------ rows longer than registers hold
// The same mathematics for rows that do not fit the registers: one block a row, which reads its operands twice (the second
// time mostly from L2: 4096 x 16384 bf16 backward 120 us; 165 us with four chunks a thread in registers, which spill).  The
// backward keeps its dw sums in shared memory, or, for rows of more than kSharedCols columns, in the partial row itself.
constexpr int kColsLimit = 1 << 30, kSharedCols = 51200;
constexpr int kLongThreads = 1024;
template <typename T, bool kShift, bool kDrop, bool kE4M3>
__global__ void __launch_bounds__(kLongThreads)
norm_fwd_long_kernel(const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ weight, float eps, Dropout d,
                     long long* __restrict__ used, T* __restrict__ h, uint32_t* __restrict__ low, T* __restrict__ out, float* __restrict__ rstd,
                     __nv_fp8_e4m3* __restrict__ q, float* __restrict__ scale, long long rows, int cols) {
  __shared__ float red[128];
  int turn = 0;
  const MaskOf<kDrop> mask(d);
  note_used(d, used);
  const int blocks = (cols + 3) / 4;
  const long long total = rows * cols;
  for (RowLoop<0> at; at.row < rows; at.row += at.step) {
    const long long base = at.row * cols;
    const int first = 8 * at.tid - (kShift ? at.offset(cols) : 0);
    auto value = [&](const Span<kShift>& s, float* v) {  // h of a chunk, unrounded
      const long long e = base + s.c0;
      Chunk<T> a = load_chunk(x + e, s, total - e);
      mask_chunk(a, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = chunk_get(a, j);
      mask.apply8(v, mask.template words_at<kShift>(at.row, blocks, s.c0));
      if (residual != nullptr) {
        Chunk<T> b = load_chunk(residual + e, s, total - e);
        mask_chunk(b, s);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += chunk_get(b, j);
      }
    };
    auto weights = [&](const Span<kShift>& s) {
      return kShift ? load_some(weight + s.c0, s.lo, s.hi) : load_chunk(weight + s.c0, s, 8);
    };
    float sq = 0.f, top = 0.f, v[8];
    for (int c = first; c < cols; c += 8 * kLongThreads) {
      const Span<kShift> s(c, cols);
      value(s, v);
      if (h != nullptr) store_chunk(h + base + c, v, s);
      if constexpr (!kE4M3 && sizeof(T) == 2) {
        if (low != nullptr && s.any()) low[low_at<kShift>(base + c, at.row)] = low_word<T>(v);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[j], v[j], sq);
      if (kE4M3) {
        if (weight != nullptr) {
          const Chunk<T> w = weights(s);
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(v[j] * chunk_get(w, j)));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(v[j]));
        }
      }
    }
    row_reduce<0, kE4M3>(sq, top, red, turn);
    const float r = weight != nullptr ? rsqrtf(sq / static_cast<float>(cols) + eps) : 1.0f;
    const RowScale by(top * r);
    if (at.tid == 0) {
      if (kE4M3) scale[at.row] = by.scale;
      else rstd[at.row] = r;
    }
    for (int c = first; c < cols; c += 8 * kLongThreads) {
      const Span<kShift> s(c, cols);
      value(s, v);
      if (weight != nullptr) {
        const Chunk<T> w = weights(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * chunk_get(w, j);
      }
      if constexpr (kE4M3) store_e4m3(q + base + c, v, by, s);
      else store_chunk(out + base + c, v, s);
    }
  }
}

// sums[0 .. 8) += v, or = v for the block's first row
template <bool kShift>
__device__ __forceinline__ void add_sums(float* sums, const float* v, const Span<kShift>& s, bool first) {
  if constexpr (!kShift) {  // 16-byte aligned
    float4* p = reinterpret_cast<float4*>(sums);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (!first) {
      a = p[0];
      b = p[1];
    }
    p[0] = make_float4(a.x + v[0], a.y + v[1], a.z + v[2], a.w + v[3]);
    p[1] = make_float4(b.x + v[4], b.y + v[5], b.z + v[6], b.w + v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= s.lo && j < s.hi) sums[j] = first ? v[j] : sums[j] + v[j];
  }
}

template <typename T, bool kShift, bool kDrop, bool kLow>
__global__ void __launch_bounds__(kLongThreads, 2)
norm_bwd_long_kernel(const T* __restrict__ dout, const T* __restrict__ dh, const T* __restrict__ h, const uint32_t* __restrict__ low,
                     const float* __restrict__ rstd, const T* __restrict__ weight, Dropout d, T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partial,
                     long long rows, int cols) {
  __shared__ float red[128];
  int turn = 0;
  const MaskOf<kDrop> mask(d);
  const int blocks = (cols + 3) / 4;
  const long long total = rows * cols;
  extern __shared__ __align__(16) float shared_sums[];
  float* out_row = partial != nullptr ? partial + static_cast<long long>(blockIdx.x) * cols : nullptr;
  bool first_row = true;
  for (RowLoop<0> at; at.row < rows; at.row += at.step, first_row = false) {
    const long long base = at.row * cols;
    const int first = 8 * at.tid - (kShift ? at.offset(cols) : 0);
    const float r = rstd[at.row];
    auto operands = [&](const Span<kShift>& s, Chunk<T>& o, Chunk<T>& hh, Chunk<T>& w) {  // and the bits below hh
      const long long e = base + s.c0;
      o = load_chunk(dout + e, s, total - e);
      hh = load_chunk(h + e, s, total - e);
      mask_chunk(o, s);
      mask_chunk(hh, s);
      w = kShift ? load_some(weight + s.c0, s.lo, s.hi) : load_chunk(weight + s.c0, s, 8);
      return LowBytes(kLow && s.any() ? low[low_at<kShift>(e, at.row)] : 0u);
    };
    auto whole = [&](const Chunk<T>& hh, const LowBytes& bits, int j) {
      if constexpr (kLow) return chunk_get_whole(hh, bits, j);
      else return chunk_get(hh, j);
    };
    float dot = 0.f, unused = 0.f, v[8];
    Chunk<T> o, hh, w;
    // a column may pass from one thread to another between rows: row_reduce's synchronisation lies between the two
    for (int c = first; c < cols; c += 8 * kLongThreads) {
      const Span<kShift> s(c, cols);
      const LowBytes bits = operands(s, o, hh, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = chunk_get(o, j) * (whole(hh, bits, j) * r);
        dot = fmaf(t, chunk_get(w, j), dot);
        v[j] = t;
      }
      if (partial != nullptr) {
        if (cols <= kSharedCols) add_sums(shared_sums + c, v, s, first_row);
        else add_sums(out_row + c, v, s, first_row);
      }
    }
    row_reduce<0, false>(dot, unused, red, turn);
    const float m = dot / static_cast<float>(cols);
    for (int c = first; c < cols; c += 8 * kLongThreads) {
      const Span<kShift> s(c, cols);
      const LowBytes bits = operands(s, o, hh, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r * (chunk_get(o, j) * chunk_get(w, j) - whole(hh, bits, j) * r * m);
      if (dh != nullptr) {
        const Chunk<T> e = load_chunk(dh + base + c, s, total - base - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += chunk_get(e, j);
      }
      if (dres != nullptr) store_chunk(dres + base + c, v, s);
      if (dx != nullptr) {
        mask.apply8(v, mask.template words_at<kShift>(at.row, blocks, s.c0));
        store_chunk(dx + base + c, v, s);
      }
    }
  }
  if (partial == nullptr || cols > kSharedCols) return;
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += kLongThreads) out_row[c] = shared_sums[c];
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

inline int check_norm_extents(int64_t rows, int64_t cols, int dtype) {
  if (cols > kColsLimit) return fail(kBadArgument, "cols must not exceed 2^30");
  return check_extents(rows, cols, dtype);
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

// How a launch covers the rows: one chunk a thread and 8, 16 or 32 lanes a row (`lanes`); or a block of `threads` a row with
// two or four chunks a thread, two as far as they reach, in exactly as many warps as the row needs; or (chunks = 0) the
// kernels for long rows.  A whole warp for rows of 64 columns: 178 us forward, 308 us backward at 2^20 rows of bf16; eight lanes:
// 84 and 122 us.
struct RowPlan {
  bool shift;
  int lanes, chunks, threads;
  int64_t grid;
};
inline RowPlan row_plan(int64_t rows, int64_t cols, int dtype, bool backward, bool drop, bool e4m3 = false) {
  RowPlan p;
  p.shift = cols % 8 != 0;
  const int64_t n = (cols + (p.shift ? 14 : 7)) / 8;  // chunks a row may touch
  p.lanes = n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 0;
  p.chunks = n <= 32 ? 1 : n <= 2 * kMaxThreads ? 2 : n <= 4 * kMaxThreads && !backward ? 4 : 0;
  p.threads = p.chunks == 1 ? kWarpBlock : p.chunks == 0 ? kLongThreads : static_cast<int>((n + 32 * p.chunks - 1) / (32 * p.chunks) * 32);
  const int64_t per_block = p.lanes != 0 ? kWarpBlock / p.lanes : 1, need = (rows + per_block - 1) / per_block;
  const int elem = dtype == 2 ? 4 : 2, regs = backward ? bwd_regs(elem, p.shift, drop, p.chunks) : fwd_regs(elem, p.shift, p.chunks, e4m3);
  const int fit = p.chunks == 0 ? (backward && cols > kSharedCols / 2 && cols <= kSharedCols ? 1 : 2) : threads_per_sm(regs) / p.threads;
  const int64_t cap = std::max(static_cast<int64_t>(sm_count()) * std::min(std::max(fit, 1), 32) / 8, int64_t{1}) * 8;  // kShift: rows advance by multiples of 8
  p.grid = std::min(need, cap);
  return p;
}
// the widest backward grid of any type, with and without dropout: each block leaves a partial row
inline int64_t most_partial_rows(int64_t rows, int64_t cols) {
  int64_t most = 0;
  for (const int dtype : {0, 1, 2})
    for (const bool drop : {false, true}) most = std::max(most, row_plan(rows, cols, dtype, true, drop).grid);
  return most;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int check_aligned(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (!aligned16(p)) return fail(kBadArgument, "matrices must be 16-byte aligned");
  return kOk;
}

template <class F>
int by_dtype(int dtype, F&& f) {
  if (dtype == 0) return f(__nv_bfloat16());
  if (dtype == 1) return f(__half());
  return f(float());
}
template <class F>
int by_flag(bool flag, F&& f) {
  return flag ? f(std::true_type()) : f(std::false_type());
}
template <int kLanes_, int kChunks_>
struct Shape {
  static constexpr int kLanes = kLanes_, kChunks = kChunks_;
};
template <bool kBackward, class F>
int by_shape(const RowPlan& p, F&& f) {
  if (p.lanes == 8) return f(Shape<8, 1>());
  if (p.lanes == 16) return f(Shape<16, 1>());
  if (p.lanes == 32) return f(Shape<32, 1>());
  if (p.chunks == 2) return f(Shape<0, 2>());
  if constexpr (!kBackward) {
    if (p.chunks == 4) return f(Shape<0, 4>());
  }
  return f(Shape<0, 0>());
}

template <bool kE4M3>
int launch_norm_fwd(const void* x, const void* residual, const void* weight, float eps, const Dropout& d, int64_t* used, void* h, void* low,
                    void* out, float* rstd, void* q, float* scale, int64_t rows, int64_t cols, int dtype, void* stream) {
  const RowPlan plan = row_plan(rows, cols, dtype, false, d.rng != nullptr, kE4M3);
  return by_dtype(dtype, [&](auto t) {
    return by_flag(plan.shift, [&](auto shift) {
      return by_flag(!kE4M3 && d.rng != nullptr, [&](auto drop) {
        return by_shape<false>(plan, [&](auto shape) {
          using T = decltype(t);
          constexpr bool kShift = decltype(shift)::value, kDrop = !kE4M3 && decltype(drop)::value;
          constexpr int kLanes = decltype(shape)::kLanes, kChunks = decltype(shape)::kChunks;
          auto kern = [] {
            if constexpr (kChunks == 0) return norm_fwd_long_kernel<T, kShift, kDrop, kE4M3>;
            else return norm_fwd_kernel<T, kShift, kDrop, kLanes, kChunks, kE4M3>;
          }();
          kern<<<static_cast<int>(plan.grid), plan.threads, 0, static_cast<cudaStream_t>(stream)>>>(
              static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), eps, d,
              reinterpret_cast<long long*>(used), static_cast<T*>(h), static_cast<uint32_t*>(low), static_cast<T*>(out), rstd, static_cast<__nv_fp8_e4m3*>(q), scale, rows,
              static_cast<int>(cols));
          return launch_check(kE4M3 ? "e4m3 rows launch" : "add_rmsnorm forward launch");
        });
      });
    });
  });
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
  rc = check_aligned({x, out});
  if (rc != kOk) return rc;
  const long long total = rows * cols, per_block = 8LL * kDropThreads * drop_unroll(dtype == 2 ? 4 : 2), need = (total + per_block - 1) / per_block;
  const long long cap = static_cast<long long>(sm_count()) * kDropBlocksPerSm;
  const int grid = static_cast<int>(need < cap ? need : cap);
  return by_dtype(dtype, [&](auto t) {
    return by_flag(d.rng != nullptr, [&](auto drop) {
      return by_flag(d.rng != nullptr && cols % 4 != 0, [&](auto shift) {
        using T = decltype(t);
        constexpr bool kDrop = decltype(drop)::value, kShift = kDrop && decltype(shift)::value;
        dropout_kernel<T, kShift, kDrop><<<grid, kDropThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), static_cast<T*>(out), total, cols, d, reinterpret_cast<long long*>(rng_used));
        return launch_check("dropout launch");
      });
    });
  });
}

extern "C" int coda_b200_add_rmsnorm_fwd(const void* x, const void* residual, const void* weight, float eps, double p, const int64_t* rng,
                                         int64_t stream_id, int64_t* rng_used, void* h, void* out, float* rstd, int64_t rows,
                                         int64_t cols, int dtype, void* stream) {
  return coda_b200_add_rmsnorm_fwd_low(x, residual, weight, eps, p, rng, stream_id, rng_used, h, nullptr, out, rstd, rows, cols, dtype, stream);
}

extern "C" int coda_b200_add_rmsnorm_fwd_low(const void* x, const void* residual, const void* weight, float eps, double p, const int64_t* rng,
                                             int64_t stream_id, int64_t* rng_used, void* h, void* h_low, void* out, float* rstd,
                                             int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_norm_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !weight || !out || !rstd) return fail(kBadArgument, "NULL pointer");
  if (h_low != nullptr && (h == nullptr || dtype == 2)) return fail(kBadArgument, "h_low goes with an h of a 2-byte type");
  rc = check_aligned({x, residual, weight, h, h_low, out});
  if (rc != kOk) return rc;
  return launch_norm_fwd<false>(x, residual, weight, eps, d, rng_used, h, h_low, out, rstd, nullptr, nullptr, rows, cols, dtype, stream);
}

extern "C" int coda_b200_rows_e4m3(const void* x, const void* residual, const void* weight, float eps, void* h, void* q, float* scale,
                                   int64_t rows, int64_t cols, int dtype, void* stream) {
  int rc = check_norm_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!x || !q || !scale) return fail(kBadArgument, "NULL pointer");
  rc = check_aligned({x, residual, weight, h, q});
  if (rc != kOk) return rc;
  const Dropout d{nullptr, 0u, 0u, 1.0f};
  return launch_norm_fwd<true>(x, residual, weight, eps, d, nullptr, h, nullptr, nullptr, nullptr, q, scale, rows, cols, dtype, stream);
}

extern "C" int64_t coda_b200_add_rmsnorm_low_bytes(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : 4 * low_words(rows, cols); }

extern "C" int64_t coda_b200_add_rmsnorm_bwd_scratch_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : most_partial_rows(rows, cols) * cols * static_cast<int64_t>(sizeof(float));
}

extern "C" int coda_b200_add_rmsnorm_bwd(const void* dout, const void* dh, const void* h, const float* rstd, const void* weight, double p,
                                         const int64_t* rng, int64_t stream_id, void* dx, void* dres, void* dweight, void* scratch,
                                         int64_t scratch_bytes, int64_t rows, int64_t cols, int dtype, void* stream) {
  return coda_b200_add_rmsnorm_bwd_low(dout, dh, h, nullptr, rstd, weight, p, rng, stream_id, dx, dres, dweight, scratch, scratch_bytes, rows,
                                       cols, dtype, stream);
}

extern "C" int coda_b200_add_rmsnorm_bwd_low(const void* dout, const void* dh, const void* h, const void* h_low, const float* rstd,
                                             const void* weight, double p, const int64_t* rng, int64_t stream_id, void* dx, void* dres,
                                             void* dweight, void* scratch, int64_t scratch_bytes, int64_t rows, int64_t cols, int dtype,
                                             void* stream) {
  int rc = check_norm_extents(rows, cols, dtype);
  if (rc != kOk) return rc;
  Dropout d;
  rc = make_dropout(p, rng, stream_id, &d);
  if (rc != kOk) return rc;
  if (rows == 0) return kOk;
  if (!dout || !h || !rstd || !weight) return fail(kBadArgument, "NULL pointer");
  if (dweight != nullptr && (scratch == nullptr || scratch_bytes < coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols)))
    return fail(kBadArgument, "the weight gradient needs coda_b200_add_rmsnorm_bwd_scratch_bytes of scratch");
  if (h_low != nullptr && dtype == 2) return fail(kBadArgument, "h_low goes with an h of a 2-byte type");
  rc = check_aligned({dout, dh, h, h_low, weight, dx, dres, scratch});
  if (rc != kOk) return rc;
  const RowPlan plan = row_plan(rows, cols, dtype, true, d.rng != nullptr);
  const int n = static_cast<int>(cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int rc2 = by_flag(plan.shift, [&](auto shift) {
      return by_flag(d.rng != nullptr, [&](auto drop) {
        return by_flag(h_low != nullptr, [&](auto bits) {
          return by_shape<true>(plan, [&](auto shape) {
            constexpr bool kShift = decltype(shift)::value, kDrop = decltype(drop)::value, kLow = sizeof(T) == 2 && decltype(bits)::value;
            constexpr int kLanes = decltype(shape)::kLanes, kChunks = decltype(shape)::kChunks;
            auto kern = [] {
              if constexpr (kChunks == 0) return norm_bwd_long_kernel<T, kShift, kDrop, kLow>;
              else return norm_bwd_kernel<T, kShift, kDrop, kLow, kLanes, kChunks>;
            }();
            int shared = 0;
            if (kChunks == 0 && dweight != nullptr && cols <= kSharedCols) {
              shared = n * static_cast<int>(sizeof(float));
              const cudaError_t e =
                  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedCols * static_cast<int>(sizeof(float)));
              if (e != cudaSuccess) return fail(kCudaError, std::string("cudaFuncSetAttribute(smem): ") + cudaGetErrorString(e));
            }
            kern<<<static_cast<int>(plan.grid), plan.threads, shared, st>>>(
                static_cast<const T*>(dout), static_cast<const T*>(dh), static_cast<const T*>(h),
                static_cast<const uint32_t*>(h_low), rstd, static_cast<const T*>(weight), d,
                static_cast<T*>(dx), static_cast<T*>(dres), dweight != nullptr ? static_cast<float*>(scratch) : nullptr, rows, n);
            return launch_check("add_rmsnorm backward launch");
          });
        });
      });
    });
    if (rc2 != kOk || dweight == nullptr) return rc2;
    fold_rows_kernel<T><<<(n + 31) / 32, 1024, 0, st>>>(static_cast<const float*>(scratch), static_cast<int>(plan.grid), n,
                                                         static_cast<T*>(dweight));
    return launch_check("add_rmsnorm weight gradient launch");
  });
}
