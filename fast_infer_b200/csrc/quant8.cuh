// 8-bit codes of cached rows: a row of 128 values x (one token, one head) is held as codes and one fp32
// scale, x ~ code * scale with scale = max|x| / Q and code = Q * x / max|x| rounded to the nearest
// code, ties to even; Q = 127 (int8) or 448 (e4m3, its largest value).
//
// Q * x is exact for x of 16 bits (11 bits times 7), and a quotient of such numbers that is not a tie
// lies further from one than half a step of fp32, so one IEEE division gives the codes of exact
// arithmetic. Both codes are exact in fp16 and bf16.
#pragma once

#include <cuda_fp8.h>

#include "umma.cuh"

namespace fi {

struct CodeI8 {
  static constexpr float kTop = 127.f;
  // codes of 4 values of at most 127
  __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const uint32_t x = (uint32_t)__float2int_rn(a) & 0xff, y = (uint32_t)__float2int_rn(b) & 0xff;
    const uint32_t z = (uint32_t)__float2int_rn(c) & 0xff, w = (uint32_t)__float2int_rn(d);
    return x | (y << 8) | (z << 16) | (w << 24);
  }
  // The same from quotients that are off by 2^-22 of themselves at most; sets `near` where one lies so close to a half that
  // its code is not sure. (1.5 * 2^23 added leaves the integer in the low bits.)
  __device__ static __forceinline__ uint32_t encode4(const float* z, bool& near) {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float shifted = __fadd_rn(z[i], 12582912.f);
      near |= fabsf(z[i] - __fsub_rn(shifted, 12582912.f)) > 0.4999f;
      t[i] = __float_as_uint(shifted);
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
  }
  // Two bytes of `v` (already offset by `bias`) as fp16: 0x64uu is 1024 + uu.
  static constexpr uint32_t kBias = 0x80808080u;  // code + 128 is the byte xor 0x80
  template <uint32_t kSel>
  __device__ static __forceinline__ uint32_t half2_of(uint32_t biased) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0x64646464, %2;" : "=r"(r) : "r"(biased), "n"(kSel));
    const __half2 m = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), m);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // fp16 pairs of codes (0, 1) and (2, 3)
  __device__ static __forceinline__ void decode4(uint32_t v, uint32_t& lo, uint32_t& hi) {
    const uint32_t b = v ^ kBias;
    lo = half2_of<0x4140>(b);
    hi = half2_of<0x4342>(b);
  }
  // The same as bf16: 0x43uu is 128 + uu for uu < 128, and 256 for uu = 128, so a code is the difference of its low
  // seven bits' number and its sign bit's.
  __device__ static __forceinline__ void decode4_bf16(uint32_t v, uint32_t& lo, uint32_t& hi) {
    uint32_t x[2];
    asm("prmt.b32 %0, %1, 0x43434343, 0x4140;" : "=r"(x[0]) : "r"(v));
    asm("prmt.b32 %0, %1, 0x43434343, 0x4342;" : "=r"(x[1]) : "r"(v));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t a = x[i] & 0xff7fff7fu, b = x[i] & 0xff80ff80u;
      const __nv_bfloat162 d =
          __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
      (i ? hi : lo) = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
};

struct CodeE4M3 {
  static constexpr float kTop = 448.f;
  __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  __device__ static __forceinline__ uint32_t encode4(const float* z, bool& near) {
    constexpr float kLess = 1.f - 0x1p-20f, kMore = 1.f + 0x1p-20f;
    const uint32_t lo = encode4(z[0] * kLess, z[1] * kLess, z[2] * kLess, z[3] * kLess);
    near |= lo != encode4(z[0] * kMore, z[1] * kMore, z[2] * kMore, z[3] * kMore);
    return lo;
  }
  __device__ static __forceinline__ void decode4(uint32_t v, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\n"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(v));
  }
};

// Codes of `v[0..N)`, a lane's part of a row whose greatest magnitude is `top`, and the row's scale. NaN or an
// infinity in the row (top then is one) gives the scale NaN and codes 0, so that every reader sees it.
template <typename C, int N>
__device__ __forceinline__ float encode_row(const float* v, float top, uint32_t* codes) {
  const bool finite = top < INFINITY;
  // Most codes are sure from a product with 1 / top; a lane that holds one that is not divides. (7742 tokens of 24 + 8
  // heads and their way back: 62 us with divisions alone, 60 so, 51 since copies run ahead of it.)
  bool near = !(top > 1e-30f && top < 1e30f);
  const float inverse = 1.f / (near ? 1.f : top);
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    float z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = v[i + j] * C::kTop * inverse;
    codes[i / 4] = C::encode4(z, near);
  }
  if (near) {
    // Q * x within fp32: a power of two off both (what that makes subnormal has the code 0 all the same)
    const float shrink = top > 1e30f ? 0x1p-20f : 1.f;
    const float den = top * shrink, num = C::kTop * shrink;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      float z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        z[j] = finite && top > 0.f ? __fdiv_rn(v[i + j] * num, den) : 0.f;
      codes[i / 4] = C::encode4(z[0], z[1], z[2], z[3]);
    }
  }
  return finite ? __fdiv_rn(top, C::kTop) : __int_as_float(0x7fffffff);
}

}  // namespace fi
