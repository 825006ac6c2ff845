// AdamW over many tensors at once.
//
//   g = coef grad,  coef = min(1, max_norm / (norm + 1e-6)), norm over all gradients
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// The tensors' pointers travel in the launch (kernel parameters), so a step uploads nothing and
// can be captured.  A launch's work is cut into chunks of one tensor each; a CTA finds its tensor
// by bisection over the chunk counts.  Memory-bound: 16-bit weights with 32-bit states move
// 22 bytes an element.
//
// 8-bit states: a block of 256 elements is held by one warp, eight elements a lane, so the
// block's largest magnitude is five shuffles.  m is held as e4m3 times a 32-bit scale.  Of v the
// root is held: it spans half the exponents, and e4m3 reaches 2^-18 of a block's largest root,
// 2^-36 of its largest v.  A root above zero stays above zero (it is rounded up to the smallest
// code), so an element whose m survives never meets a denominator of eps alone.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.h"

namespace tcpxb_train {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;
constexpr float kE4m3Max = 448.f;

template <int N> struct List {
  tcpxbAdamwTensor t[N];
  unsigned end[N];  // chunks up to and with tensor i
  int count, first;  // `first`: number of t[0] in the caller's list
};
// Two sizes of the same launch: a short list does not pay for copying 30 KB of parameters.
using Short = List<24>;
using Long = List<380>;

struct Rates {
  float stepSize, rootCorrection;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};
struct Scratch {
  float coef;
  float pad;
  Rates rates[1];
};

template <class L> __device__ __forceinline__ int tensorOf(const L& l, unsigned chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (chunk < l.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Counts every tensor's step and takes what depends on it, in 64 bits: 1 - b^t cancels.
template <class L> __global__ void prepareKernel(const __grid_constant__ L l, const tcpxbAdamw a) {
  auto* s = static_cast<Scratch*>(a.scratch);
  if (threadIdx.x == 0 && l.first == 0) {
    float coef = 1.f;
    if (a.grad_norm) {
      const float c = a.max_norm / (*a.grad_norm + 1e-6f);
      coef = c < 1.f || c != c ? c : 1.f;
    }
    s->coef = coef;
  }
  for (int i = threadIdx.x; i < l.count; i += blockDim.x) {
    const int t = ++*l.t[i].step;
    s->rates[l.first + i].stepSize = float(double(a.lr) / (1.0 - pow(double(a.beta1), t)));
    s->rates[l.first + i].rootCorrection = float(1.0 / sqrt(1.0 - pow(double(a.beta2), t)));
  }
}

struct Step {
  float beta1, beta2, eps, keep, stepSize, rootCorrection, coef;
  __device__ __forceinline__ float operator()(float p, float g, float& m, float& v) const {
    g *= coef;
    m = m * beta1 + (1.f - beta1) * g;
    v = v * beta2 + (1.f - beta2) * g * g;
    return p * keep - stepSize * m / (sqrtf(v) * rootCorrection + eps);
  }
};

__device__ __forceinline__ float fromE4m3(__nv_fp8_storage_t x) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3))); }

// Largest magnitude of the warp; NaN is left out (its code is NaN by itself).
__device__ __forceinline__ float warpTop(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

template <class T, class L, bool kSmall> __global__ void __launch_bounds__(kThreads) stepKernel(const __grid_constant__ L l, const tcpxbAdamw a) {
  const int i = tensorOf(l, blockIdx.x);
  const tcpxbAdamwTensor& t = l.t[i];
  const long long begin = (long long)(blockIdx.x - (i ? l.end[i - 1] : 0)) * kChunk;
  const long long end = min((long long)t.n, begin + kChunk);
  const auto* s = static_cast<const Scratch*>(a.scratch);
  const Step step{a.beta1, a.beta2, a.eps, 1.f - a.lr * a.weight_decay, s->rates[l.first + i].stepSize, s->rates[l.first + i].rootCorrection, s->coef};
  T* p = static_cast<T*>(t.p);
  const T* g = static_cast<const T*>(t.g);
  if (!kSmall) {
    float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
    for (long long e = begin + threadIdx.x; e < end; e += kThreads) {
      float mm = m[e], vv = v[e];
      const float w = step(t.master ? t.master[e] : toFloat(p[e]), toFloat(g[e]), mm, vv);
      m[e] = mm, v[e] = vv, p[e] = fromFloat<T>(w);
      if (t.master) t.master[e] = w;
    }
    return;
  }
  auto *m = static_cast<__nv_fp8_storage_t*>(t.m), *v = static_cast<__nv_fp8_storage_t*>(t.v);
  const int lane = threadIdx.x % 32;
  for (long long b = begin + threadIdx.x / 32 * TCPXB_ADAMW_BLOCK; b < end; b += kThreads / 32 * TCPXB_ADAMW_BLOCK) {
    const long long block = b / TCPXB_ADAMW_BLOCK;
    const float ms = t.m_scale[block], vs = t.v_scale[block];
    float mm[8] = {}, vv[8] = {}, topM = 0.f, topV = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const long long e = b + k * 32 + lane;
      if (e >= end) continue;
      mm[k] = fromE4m3(m[e]) * ms;
      const float root = fromE4m3(v[e]) * vs;
      vv[k] = root * root;
      const float w = step(t.master ? t.master[e] : toFloat(p[e]), toFloat(g[e]), mm[k], vv[k]);
      p[e] = fromFloat<T>(w);
      if (t.master) t.master[e] = w;
      vv[k] = sqrtf(vv[k]);
      topM = fmaxf(topM, fabsf(mm[k])), topV = fmaxf(topV, vv[k]);
    }
    topM = warpTop(topM), topV = warpTop(topV);
    // below 1e-30 a block is held as zeros: the factor back would leave the range
    const float toM = topM >= 1e-30f ? kE4m3Max / topM : 0.f, toV = topV >= 1e-30f ? kE4m3Max / topV : 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const long long e = b + k * 32 + lane;
      if (e >= end) continue;
      float root = vv[k] * toV;
      if (root > 0.f) root = fmaxf(root, 0.001953125f);  // 2^-9, the smallest code above zero
      m[e] = __nv_cvt_float_to_fp8(mm[k] * toM, __NV_SATFINITE, __NV_E4M3);
      v[e] = __nv_cvt_float_to_fp8(root, __NV_SATFINITE, __NV_E4M3);
    }
    if (lane == 0) {
      t.m_scale[block] = topM >= 1e-30f ? topM / kE4m3Max : 0.f;
      t.v_scale[block] = topV >= 1e-30f ? topV / kE4m3Max : 0.f;
    }
  }
}

__device__ __forceinline__ double blockSum(double x) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = x;
  __syncthreads();
  x = 0;
  for (int i = 0; i < int(blockDim.x) / 32; i++) x += part[i];
  return x;
}

template <class T, class L> __global__ void __launch_bounds__(kThreads) squaresKernel(const __grid_constant__ L l, double* partial) {
  const int i = tensorOf(l, blockIdx.x);
  const long long begin = (long long)(blockIdx.x - (i ? l.end[i - 1] : 0)) * kChunk;
  const long long end = min((long long)l.t[i].n, begin + kChunk);
  const T* g = static_cast<const T*>(l.t[i].g);
  float sum = 0.f;  // 32 squares a thread
  for (long long e = begin + threadIdx.x; e < end; e += kThreads) {
    const float x = toFloat(g[e]);
    sum += x * x;
  }
  const double all = blockSum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = all;
}

__global__ void normKernel(const double* partial, long long n, float* norm) {
  double sum = 0;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) sum += partial[i];
  sum = blockSum(sum);
  if (threadIdx.x == 0) *norm = float(sqrt(sum));
}

long long chunksOf(const tcpxbAdamwTensor& t) { return (t.n + kChunk - 1) / kChunk; }

// Calls f(list, chunks) for the tensors in lists of at most N, leaving out those without elements.
template <class L, int N, class F> int inLists(const tcpxbAdamwTensor* tensors, int count, F f) {
  static thread_local L l;
  for (int first = 0; first < count;) {
    long long chunks = 0;
    l.count = 0, l.first = first;
    int i = first;
    for (; i < count && l.count < N && chunks + chunksOf(tensors[i]) < (1ll << 31); i++) {
      l.t[l.count] = tensors[i];
      chunks += chunksOf(tensors[i]);
      l.end[l.count++] = unsigned(chunks);
    }
    if (const int rc = f(l, chunks)) return rc;
    first = i;
  }
  return TCPXB_T_OK;
}
template <class F> int inLists(const tcpxbAdamwTensor* tensors, int count, F f) {
  return count <= 24 ? inLists<Short, 24>(tensors, count, f) : inLists<Long, 380>(tensors, count, f);
}

int check(const tcpxbAdamwTensor* t, int count, int dtype, bool step, int bits) {
  if (count < 0 || (count && !t)) return fail(TCPXB_T_INVALID, "null list");
  if (dtype != TCPXB_T_BF16 && dtype != TCPXB_T_F16 && dtype != TCPXB_T_F32) return fail(TCPXB_T_INVALID, "unknown type %d", dtype);
  for (int i = 0; i < count; i++) {
    if (t[i].n < 0 || t[i].n > (1ll << 43)) return fail(TCPXB_T_INVALID, "tensor %d has a bad size", i);
    if (t[i].n && !t[i].g) return fail(TCPXB_T_INVALID, "tensor %d has no gradient", i);
    if (!step) continue;
    if (!t[i].step || (t[i].n && (!t[i].p || !t[i].m || !t[i].v || (bits == 8 && (!t[i].m_scale || !t[i].v_scale)))))
      return fail(TCPXB_T_INVALID, "tensor %d lacks its weights, states, scales or step", i);
  }
  return TCPXB_T_OK;
}

template <class T> int step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw& a, cudaStream_t s) {
  return inLists(tensors, count, [&](const auto& l, long long chunks) {
    using L = std::decay_t<decltype(l)>;
    prepareKernel<<<1, l.count <= 128 ? 128 : 384, 0, s>>>(l, a);
    if (const int rc = launched("adamw, rates")) return rc;
    if (!chunks) return int(TCPXB_T_OK);
    if (a.state_bits == 8) stepKernel<T, L, true><<<unsigned(chunks), kThreads, 0, s>>>(l, a);
    else stepKernel<T, L, false><<<unsigned(chunks), kThreads, 0, s>>>(l, a);
    return launched("adamw");
  });
}

template <class T> int squares(const tcpxbAdamwTensor* tensors, int count, float* norm, double* partial, cudaStream_t s) {
  long long done = 0;
  const int rc = inLists(tensors, count, [&](const auto& l, long long chunks) {
    using L = std::decay_t<decltype(l)>;
    if (!chunks) return int(TCPXB_T_OK);
    squaresKernel<T, L><<<unsigned(chunks), kThreads, 0, s>>>(l, partial + done);
    done += chunks;
    return launched("gradient norm");
  });
  if (rc) return rc;
  normKernel<<<1, 1024, 0, s>>>(partial, done, norm);
  return launched("gradient norm, sum");
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" size_t tcpxb_adamw_scratch_bytes(int count) { return sizeof(Scratch) + sizeof(Rates) * size_t(count > 0 ? count : 0); }

extern "C" int tcpxb_adamw_step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw* a, void* stream) {
  if (!a || !a->scratch) return fail(TCPXB_T_INVALID, "null argument");
  if (a->state_bits != 8 && a->state_bits != 32) return fail(TCPXB_T_INVALID, "states have 8 or 32 bits, not %d", a->state_bits);
  if (const int rc = check(tensors, count, a->dtype, true, a->state_bits)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == TCPXB_T_BF16) return step<__nv_bfloat16>(tensors, count, *a, s);
  if (a->dtype == TCPXB_T_F16) return step<__half>(tensors, count, *a, s);
  return step<float>(tensors, count, *a, s);
}

extern "C" size_t tcpxb_grad_norm_scratch_bytes(const tcpxbAdamwTensor* tensors, int count) {
  long long chunks = 0;
  for (int i = 0; tensors && i < count; i++) chunks += chunksOf(tensors[i]);
  return sizeof(double) * size_t(chunks + 1);
}

extern "C" int tcpxb_grad_norm(const tcpxbAdamwTensor* tensors, int count, int dtype, float* norm, void* scratch, void* stream) {
  if (!norm || !scratch) return fail(TCPXB_T_INVALID, "null argument");
  if (const int rc = check(tensors, count, dtype, false, 32)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  auto* partial = static_cast<double*>(scratch);
  if (dtype == TCPXB_T_BF16) return squares<__nv_bfloat16>(tensors, count, norm, partial, s);
  if (dtype == TCPXB_T_F16) return squares<__half>(tensors, count, norm, partial, s);
  return squares<float>(tensors, count, norm, partial, s);
}
