// What the training kernels share: types, errors, vectors of eight elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tcpxb/train.h"

namespace tcpxb_train {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// The last launch's status, as a return value.
int launched(const char* what);

template <class T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float toFloat(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T fromFloat(float x);
template <> __device__ __forceinline__ float fromFloat<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float x) { return __float2half_rn(x); }

// Eight elements on a 16-byte boundary (fp32: 32 bytes as two such vectors).
template <class T> struct alignas(16) Vec8 { T x[8]; };

template <class T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  const Vec8<T> v = *reinterpret_cast<const Vec8<T>*>(p);
#pragma unroll
  for (int i = 0; i < 8; i++) f[i] = toFloat(v.x[i]);
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < 8; i++) v.x[i] = fromFloat<T>(f[i]);
  *reinterpret_cast<Vec8<T>*>(p) = v;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
inline bool headsOk(const tcpxbHeads& h, int elemBytes) {
  const int64_t per = 16 / elemBytes;
  return h.ptr && reinterpret_cast<uintptr_t>(h.ptr) % 16 == 0 && h.stride_b % per == 0 && h.stride_s % per == 0 && h.stride_h % per == 0;
}

}  // namespace tcpxb_train
