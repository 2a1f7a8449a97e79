// vec.cuh -- 16-byte vectors of fp32 / fp16 / bf16 elements, and rows that begin
// on any element.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sinkslot {

template <typename T>
struct Vec16 {
  static constexpr int N = 16 / (int)sizeof(T);
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// The elements of a 16-byte vector as fp32 and back (one rounding each).
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4], const float*) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], const __half*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], const float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __half*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __nv_bfloat16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two floats in one 64-bit register and the arithmetic that sm_100 has on them.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 parts(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The largest element of a vector (NaNs count as nothing: the sum shows them).
__device__ __forceinline__ float max_of(const uint4& u, const float*) {
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
               fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
__device__ __forceinline__ float max_of(const uint4& u, const __half*) {
  const __half2 a = __hmax2(*reinterpret_cast<const __half2*>(&u.x),
                            *reinterpret_cast<const __half2*>(&u.y));
  const __half2 b = __hmax2(*reinterpret_cast<const __half2*>(&u.z),
                            *reinterpret_cast<const __half2*>(&u.w));
  const float2 t = __half22float2(__hmax2(a, b));
  return fmaxf(t.x, t.y);
}
__device__ __forceinline__ float max_of(const uint4& u, const __nv_bfloat16*) {
  const __nv_bfloat162 a = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&u.x),
                                   *reinterpret_cast<const __nv_bfloat162*>(&u.y));
  const __nv_bfloat162 b = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&u.z),
                                   *reinterpret_cast<const __nv_bfloat162*>(&u.w));
  const float2 t = __bfloat1622float2(__hmax2(a, b));
  return fmaxf(t.x, t.y);
}

// A row of n elements from p: `head` elements up to the first 16-byte boundary,
// `body` whole vectors, then the rest.
struct RowSpan {
  int64_t head, body;
};
template <typename T>
__device__ __forceinline__ RowSpan row_span(const T* p, int64_t n) {
  const int64_t off = (int64_t)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  int64_t head = off ? Vec16<T>::N - off : 0;
  if (head > n) head = n;
  return {head, (n - head) / Vec16<T>::N};
}

// 2^x, good to about 2^-22 of its value (results under 2^-126 flush to zero: they
// are nothing next to a row's largest term, 1).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace sinkslot
