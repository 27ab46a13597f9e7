// Block-scaled key/value cache: the host-side checks, row addressing and 8-bit
// codes that the append, decode and evict kernels share.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace pa {

// Element kinds of a cache (template parameter of every kernel).
enum : int { kCacheF16 = 0, kCacheBF16 = 1, kCacheE4M3 = 2, kCacheI8 = 3 };

// Division of 0 <= n < 2^31 by a fixed d >= 1 as a high product, an add and a shift
// (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};

inline FastDiv make_fastdiv(uint32_t d) {
  uint32_t s = 0;
  while (s < 31 && (1u << s) < d) ++s;
  const uint64_t m = ((1ull << 32) * ((1ull << s) - d)) / d + 1;
  return {d, static_cast<uint32_t>(m), s};
}

#if defined(__CUDACC__)
__device__ __forceinline__ int fast_div(const FastDiv& f, int n) {
  const uint32_t u = static_cast<uint32_t>(n);
  return static_cast<int>((__umulhi(u, f.mul) + u) >> f.shift);
}
#endif

// What the kernels need of a checked descriptor. Strides are in bytes for the
// cache and in elements for scales and per-row arrays.
struct CacheView {
  int64_t key_stride, head_stride, page_stride;
  int64_t scale_head, scale_page;
  int64_t row_head, row_seq;
  int32_t B, Hq, Hkv, D;
  int32_t page_size, num_pages, max_pages, scale_block, max_len;
  int32_t kind;
  int32_t q_bf16;
  int32_t paged;
  FastDiv by_page, by_block;
};

// Which optional parts of a descriptor a call uses.
struct CacheUse {
  bool paged;
  bool rows;    // a per-row array (weights, positions) is passed
  bool decode;  // queries: head groups and the softmax scale matter
};

// Checks `d` for a call and fills `v` (csrc/cache_append.cu).
pa_status check_cache(const pa_block_cache_desc* d, const CacheUse& use, CacheView* v,
                      const char* who);
// Checks the cache's pointers: non-null, aligned, scales exactly where they belong.
pa_status check_cache_ptrs(const CacheView& v, const void* k, const void* v_cache,
                           const void* k_scales, const void* v_scales, const char* who);

#if defined(__CUDACC__)

__host__ __device__ constexpr bool cache_8bit(int kind) { return kind >= kCacheE4M3; }
__host__ __device__ constexpr int cache_esz(int kind) { return cache_8bit(kind) ? 1 : 2; }

// Page of row `row` of sequence `b`, or -1 (reported) for an entry outside the cache.
__device__ __forceinline__ int32_t cache_page(const CacheView& v, const int32_t* table, int b, int row,
                                              int* status) {
  if (!table) return b;
  const int32_t page = table[static_cast<int64_t>(b) * v.max_pages + fast_div(v.by_page, row)];
  if (page < 0 || page >= v.num_pages) {
    atomicExch(status, kStatusBadPage);
    return -1;
  }
  return page;
}

// Place of a row inside its page.
__device__ __forceinline__ int cache_at(const CacheView& v, int row) {
  return v.paged ? row - fast_div(v.by_page, row) * v.page_size : row;
}

__device__ __forceinline__ int64_t cache_row(const CacheView& v, int32_t page, int h, int at) {
  return page * v.page_stride + h * v.head_stride + at * v.key_stride;
}

__device__ __forceinline__ int64_t cache_scale(const CacheView& v, int32_t page, int h, int at) {
  return page * v.scale_page + h * v.scale_head + fast_div(v.by_block, at);
}

// The least power of two s with amax <= qmax * s, at least 2^-100, by exponent
// arithmetic: amax = m * 2^e with m in [1, 2), qmax = 1.75 * 2^8 (e4m3) or
// 1.984375 * 2^6 (int8), both exact.
template <int KIND>
__device__ __forceinline__ float cache_need_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = static_cast<int>(bits >> 23) - 127;
  const uint32_t man = bits & 0x7fffffu;
  constexpr uint32_t top = KIND == kCacheE4M3 ? 0x600000u : 0x7e0000u;  // mantissa of qmax
  e += (man > top ? 1 : 0) - (KIND == kCacheE4M3 ? 8 : 6);
  e = e < -100 ? -100 : e;  // also zero and subnormal magnitudes
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two 8-bit codes (low byte first) as floats.
template <int KIND>
__device__ __forceinline__ float2 cache_dec2(uint32_t two) {
  if (KIND == kCacheE4M3) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
  }
  return make_float2(static_cast<float>(static_cast<int8_t>(two & 0xff)),
                     static_cast<float>(static_cast<int8_t>((two >> 8) & 0xff)));
}

// Nearest 8-bit codes of two floats, ties to even, saturating (low byte first).
template <int KIND>
__device__ __forceinline__ uint32_t cache_enc2(float a, float b) {
  if (KIND == kCacheE4M3)
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  int x = __float2int_rn(a), y = __float2int_rn(b);  // NaN gives 0
  x = x > 127 ? 127 : (x < -127 ? -127 : x);
  y = y > 127 ? 127 : (y < -127 ? -127 : y);
  return static_cast<uint32_t>(x & 0xff) | (static_cast<uint32_t>(y & 0xff) << 8);
}

// Largest finite magnitude of amax and x (NaN and infinities are passed over).
__device__ __forceinline__ float cache_amax(float amax, float x) {
  const float m = fabsf(x);
  return m < INFINITY ? fmaxf(amax, m) : amax;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Largest finite magnitude among 16 codes. Magnitudes compare as integers, two
// 16-bit lanes at a time (a lane's high byte decides); only a NaN among them needs
// a closer look.
template <int KIND>
__device__ __forceinline__ float cache_absmax(const uint4& q) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t odd = 0u, even = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x = w[i];
    if (KIND == kCacheI8) {
      const uint32_t neg = (x >> 7) & 0x01010101u;
      x = (x ^ (neg * 0xffu)) + neg;  // |-128| is 0x80 and carries nowhere
    } else {
      x &= 0x7f7f7f7fu;
    }
    odd = max_u16x2(odd, x);
    even = max_u16x2(even, __byte_perm(x, 0u, 0x2404));
  }
  const uint32_t m = max_u16x2(odd, even);
  const uint32_t top = (m >> 24) > ((m >> 8) & 0xffu) ? m >> 24 : (m >> 8) & 0xffu;
  if (KIND == kCacheI8) return static_cast<float>(top);
  if (top != 0x7fu) return cache_dec2<KIND>(top).x;
  float f = 0.f;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) f = cache_amax(f, cache_dec2<KIND>((w[i >> 2] >> (8 * (i & 3))) & 0xffu).x);
  return f;
}

// Whether from / to is a power of two from 2^-14 to 2^15: codes then move between
// the scales in fp16 arithmetic that rounds once.
__device__ __forceinline__ bool cache_easy_ratio(float from, float to) {
  const uint32_t a = __float_as_uint(from), b = __float_as_uint(to);
  const int k = static_cast<int>(a >> 23) - static_cast<int>(b >> 23);
  return ((a | b) & 0x807fffffu) == 0u && a != 0u && b != 0u && k >= -14 && k <= 15;
}

// Four fp16 values as e4m3 codes (first in the low byte), and four codes as fp16.
__device__ __forceinline__ uint32_t e4m3_from_h4(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f16x2 l, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 h, %2;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(d)
      : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void e4m3_to_h4(uint32_t w, uint32_t& a, uint32_t& b) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(a), "=r"(b)
      : "r"(w));
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, __half2 b) {
  const __half2 p = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// That ratio, twice.
__device__ __forceinline__ __half2 cache_ratio(float from, float to) {
  const uint32_t k = (__float_as_uint(from) >> 23) - (__float_as_uint(to) >> 23) + 15u;
  const uint32_t h = (k << 10) | (k << 26);
  return *reinterpret_cast<const __half2*>(&h);
}

// Four codes times such a ratio, as codes. int8: 1536 + x rounds x to an integer
// whose low byte is the code; products stay within the format where the new scale
// fits them.
template <int KIND>
__device__ __forceinline__ uint32_t cache_rescale4(uint32_t w, __half2 ratio) {
  if (KIND == kCacheE4M3) {
    uint32_t a, b;
    e4m3_to_h4(w, a, b);
    return e4m3_from_h4(h2_mul(a, ratio), h2_mul(b, ratio));
  }
  const uint32_t u = w ^ 0x80808080u;  // value + 128
  const __half2 bias = __floats2half2_rn(1152.f, 1152.f), magic = __floats2half2_rn(1536.f, 1536.f);
  uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);  // 1024 + that
  const __half2 a = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&lo), bias), ratio, magic);
  const __half2 b = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&hi), bias), ratio, magic);
  return __byte_perm(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b), 0x6420);
}

template <bool BF16>
__device__ __forceinline__ float2 cache_unpack(uint32_t w) {
  if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

#endif  // __CUDACC__

}  // namespace pa
