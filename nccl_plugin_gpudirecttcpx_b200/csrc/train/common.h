// What the training kernels share: types, errors, vectors of eight elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tcpxb/train.h"

namespace tcpxb_train {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Makes the tensors' device the thread's.  A thread that only autograd has used so far has a device but
// no context, which the driver's calls need; this gives it both.
int use(int device);
// The last launch's status, as a return value.
int launched(const char* what);

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float toFloat(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T fromFloat(float x);
template <> __device__ __forceinline__ float fromFloat<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float x) { return __float2half_rn(x); }

// Eight elements on a 16-byte boundary (fp32: 32 bytes as two such vectors).
template <class T> struct alignas(16) Vec8 { T x[8]; };

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A lane's eight elements as four pairs, and back, rounded; two 16-bit elements share a register.
__device__ __forceinline__ float2 unpack2(uint32_t x, __nv_bfloat16) { return {__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)}; }
__device__ __forceinline__ float2 unpack2(uint32_t x, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
template <class T> __device__ __forceinline__ void pairs(const Vec8<T>& v, float2 (&f)[4]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 w = *reinterpret_cast<const uint4*>(&v);
    f[0] = unpack2(w.x, T()), f[1] = unpack2(w.y, T()), f[2] = unpack2(w.z, T()), f[3] = unpack2(w.w, T());
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = {v.x[2 * i], v.x[2 * i + 1]};
  }
}
template <class T> __device__ __forceinline__ Vec8<T> rounded(const float2 (&f)[4]) {
  Vec8<T> v;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(&v) = {pack2<T>(f[0].x, f[0].y), pack2<T>(f[1].x, f[1].y), pack2<T>(f[2].x, f[2].y), pack2<T>(f[3].x, f[3].y)};
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v.x[2 * i] = f[i].x, v.x[2 * i + 1] = f[i].y;
  }
  return v;
}

// A kernel behind another one of the same call may be set up while that one ends, and waits here until
// all of its writes are there.  It may be set up once all blocks of the one before have called
// letNextStart(), or have ended: then it takes the room that they leave.  In turn with and without on one GPU:
// 7 us of a pass of attention both ways over 4 x 2048 tokens, 32/8 heads of 64 (1.7 %; 440 us where this was not
// compared, by the clock), 6 us of an AdamW step over 323 M weights with clipping (1170 us).  A call's first kernel is launched in the ordinary way, behind all that stands in the stream.
__device__ __forceinline__ void waitForPrevious() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void letNextStart() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class K, class... A> int launchBehind(bool own, K* kernel, dim3 grid, int threads, size_t shared, cudaStream_t s, const char* what, const A&... args) {
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid, config.blockDim = dim3(threads), config.dynamicSmemBytes = shared, config.stream = s;
  config.attrs = &attribute, config.numAttrs = own ? 1 : 0;
  cudaLaunchKernelEx(&config, kernel, args...);
  return launched(what);
}

inline bool headsOk(const tcpxbHeads& h, int elemBytes) {
  const int64_t per = 16 / elemBytes;
  return h.ptr && reinterpret_cast<uintptr_t>(h.ptr) % 16 == 0 && h.stride_b % per == 0 && h.stride_s % per == 0 && h.stride_h % per == 0;
}

}  // namespace tcpxb_train
