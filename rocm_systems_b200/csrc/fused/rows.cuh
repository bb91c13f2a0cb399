// Small device helpers of the kernels that work on rows of bf16 values with fp32 arithmetic.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {
namespace rows {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2Fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in a 64-bit register: one instruction for both.
typedef unsigned long long F2;
__device__ __forceinline__ F2 makeF2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void splitF2(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fmaF2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mulF2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 addF2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 exp2F2(F2 x) {
  float a, b;
  splitF2(x, a, b);
  return makeF2(exp2Fast(a), exp2Fast(b));
}
// 2^x without the special-function unit, whose 16 results per clock and SM are what a softmax runs out of first: x = n + f with n the nearest
// whole number (added and taken off again at a scale where fp32 has no fraction left), 2^f for |f| <= 1/2 by the polynomial of degree 4
// with the smallest largest relative error (2.7e-6 in fp32; Remez exchange), times 2^n, whose bits n is shifted into. Below -126 the result is 2^-126. A NaN
// stays one by that product (n added to the exponent's bits made it the largest finite number).
__device__ __forceinline__ F2 exp2Poly(F2 x) {
  float a, b;
  splitF2(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-126.f));
  x = makeF2(a, b);
  const auto both = [](float v) { return makeF2(v, v); };
  const F2 n = addF2(x, both(12582912.f));  // 1.5 * 2^23
  const F2 f = fmaF2(addF2(n, both(-12582912.f)), both(-1.f), x);
  F2 p = fmaF2(both(0.009570102207362652f), f, both(0.05591785907745361f));
  p = fmaF2(p, f, both(0.240247443318367f));
  p = fmaF2(p, f, both(0.6931217908859253f));
  p = fmaF2(p, f, both(0.9999992847442627f));
  splitF2(n, a, b);
  return mulF2(p, makeF2(__int_as_float((__float_as_int(a) << 23) + 0x3f800000), __int_as_float((__float_as_int(b) << 23) + 0x3f800000)));
}
// Two bf16 values of a 32-bit word.
__device__ __forceinline__ F2 unpackF2(uint32_t w) { return makeF2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Sum / maximum over groups of N consecutive lanes (N a power of two); every lane gets the result.
template <int N> __device__ __forceinline__ float laneSum(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int N> __device__ __forceinline__ float laneMax(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ void unpack4(const uint2& p, float (&f)[4]) {
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.y));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(F2 v) {
  float a, b;
  splitF2(v, a, b);
  return pack2(a, b);
}
__device__ __forceinline__ uint2 pack4(const float (&f)[4]) { return make_uint2(pack2(f[0], f[1]), pack2(f[2], f[3])); }
__device__ __forceinline__ void unpack8(const uint4& p, float (&f)[8]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) { return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])); }

// 16 packed words (32 bf16 values) of a row to global memory: in 32-byte pieces where `wide` (the address is on a 32-byte boundary), whole
// sectors although every lane of a warp has a row of its own, else in 16-byte pieces; `words` of them exist (a multiple of 4, and of 8 where wide).
__device__ __forceinline__ void storeRow16(__nv_bfloat16* dst, const uint32_t (&w)[16], int words, bool wide) {
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    if (wide) {
      if (i < words)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 2 * i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                     "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                     : "memory");
    } else {
      if (i < words) *reinterpret_cast<uint4*>(dst + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      if (i + 4 < words) *reinterpret_cast<uint4*>(dst + 2 * i + 8) = make_uint4(w[i + 4], w[i + 5], w[i + 6], w[i + 7]);
    }
  }
}

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store(float* p, float x) { *p = x; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }

}  // namespace rows
}  // namespace b200
