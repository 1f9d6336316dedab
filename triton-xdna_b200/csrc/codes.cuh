// 8-bit codes of a KV cache's head vectors.  A vector of bf16 numbers whose
// largest magnitude is a has the exponent e, the smallest whole number with a <=
// M 2^e (M = 127 for int8, 448 for e4m3), and the codes rne(x 2^-e); a code c
// stands for c 2^e.  e is kept as the byte e + 127.  The scale is a power of two, so
// what a code stands for is a bf16 number: reading back rounds nothing, and a
// matrix product sees exactly what is stored.  It costs int8 up to one of its
// seven bits (a scale of a / 127 would use them all) and e4m3 nothing.
// Bytes: 47 (so that sums of 2^-e stay inside fp32, see kShareUp in paged.cu;
// smaller vectors round to zeros, and zeros have it) to 248 / 246 (what the largest codes stand for is finite;
// vectors beyond saturate), and 255: an infinity or NaN in the vector, which
// reads as NaN throughout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace xb {
namespace codes {

constexpr int kLeastByte = 47, kNanByte = 255;

// Format of a cache's pages (template argument of the kernels that serve all three)
enum Format : int { kBf16 = 0, kInt8 = 1, kE4m3 = 2 };

// The exponent byte of a vector whose largest magnitude has the bf16 bits `top`.
// a = (1 + f / 128) 2^(top / 128 - 127) with f = top % 128: 127 = (1 + 126 / 128) 2^6,
// 448 = (1 + 96 / 128) 2^8.
template <Format F>
__device__ __forceinline__ int exponent_byte(uint32_t top) {
  constexpr int bits = F == kInt8 ? 6 : 8, fraction = F == kInt8 ? 126 : 96, last = F == kInt8 ? 248 : 246;
  if (top >= 0x7f80u) return kNanByte;
  const int b = (int)(top >> 7) - bits + ((int)(top & 127u) > fraction);
  return min(max(b, kLeastByte), last);
}

// 2^e of a byte (NaN for 255), and 2^-e (0 for 255)
__device__ __forceinline__ float byte_scale(int b) {
  return b == kNanByte ? __int_as_float(0x7fc00000) : __int_as_float(b << 23);
}
__device__ __forceinline__ float byte_inverse(int b) {
  return b == kNanByte ? 0.0f : __int_as_float((254 - b) << 23);
}

// Eight codes of x 2^-e (x: eight bf16 numbers in 32-bit words), |x 2^-e| < 128.5 or 512.
template <Format F>
__device__ __forceinline__ uint2 encode8(const uint4& x, float inverse) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t r[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = __uint_as_float(w[2 * h + i] << 16);
      v[2 * i + 1] = __uint_as_float(w[2 * h + i] & 0xffff0000u);
    }
    if constexpr (F == kInt8) {
      // 1.5 2^23 more, a number's last byte is the nearest whole number's, to even in the middle
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(v[i], inverse, 12582912.0f));
      r[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * inverse), "f"(v[0] * inverse));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * inverse), "f"(v[2] * inverse));
      r[h] = (uint32_t)lo | (uint32_t)hi << 16;
    }
  }
  return make_uint2(r[0], r[1]);
}

// Two e4m3 codes as fp16 (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

// Four codes in a register as fp16 pairs (exact): bytes 0 and 2, bytes 1 and 3.
// int8: the byte c + 128 (the sign bit flipped) in the low bits of 1024 is 1152 + c.
template <Format F>
__device__ __forceinline__ void to_half2(uint32_t v, uint32_t& even, uint32_t& odd) {
  if constexpr (F == kInt8) {
    v ^= 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    const uint32_t m0 = __byte_perm(v, 0x64646464u, 0x4240), m1 = __byte_perm(v, 0x64646464u, 0x4341);
    const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&m0), bias);
    const __half2 h1 = __hsub2(*reinterpret_cast<const __half2*>(&m1), bias);
    even = *reinterpret_cast<const uint32_t*>(&h0);
    odd = *reinterpret_cast<const uint32_t*>(&h1);
  } else {
    v = __byte_perm(v, 0, 0x3120);
    even = e4m3x2_to_half2((uint16_t)v);
    odd = e4m3x2_to_half2((uint16_t)(v >> 16));
  }
}

// What four codes stand for, as bf16 (exact)
template <Format F>
__device__ __forceinline__ uint2 decode4(uint32_t v, float scale) {
  float x[4];
  if constexpr (F == kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(v >> (8 * i));
  } else {
    const uint32_t lo = e4m3x2_to_half2((uint16_t)v), hi = e4m3x2_to_half2((uint16_t)(v >> 16));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
  const __nv_bfloat162 p = __floats2bfloat162_rn(x[0] * scale, x[1] * scale);
  const __nv_bfloat162 q = __floats2bfloat162_rn(x[2] * scale, x[3] * scale);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
}

}  // namespace codes
}  // namespace xb
