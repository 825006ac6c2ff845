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
// block's largest magnitude is one instruction.  m is held as e4m3 times a 32-bit scale.  Of v the
// root is held: it spans half the exponents, and e4m3 reaches 2^-18 of a block's largest root,
// 2^-36 of its largest v.  A root above zero stays above zero (it is rounded up to the smallest
// code), so an element whose m survives never meets a denominator of eps alone.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.h"

namespace tcpxb_train {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // elements of a CTA (32768: 1213 us instead of 1167 us for 323 M weights with clipping)
constexpr float kE4m3Max = 448.f, kLeastCode = 0.001953125f;  // the largest code, and 2^-9, the smallest above zero

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

__device__ __forceinline__ float rootOfSum(const double* partial, long long n) {
  double sum = 0;
  for (long long i0 = threadIdx.x; i0 < n; i0 += 8 * blockDim.x) {
    double x[8];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = i0 + k * blockDim.x < n ? partial[i0 + k * blockDim.x] : 0.0;
#pragma unroll
    for (int k = 0; k < 8; k++) sum += x[k];
  }
  return float(sqrt(blockSum(sum)));
}

// Counts every tensor's step and takes what depends on it, in 64 bits: 1 - b^t cancels.  The first
// list's launch also takes the norm out of `partials` sums, where it is computed here.
template <class L> __global__ void __launch_bounds__(1024) prepareKernel(const __grid_constant__ L l, const tcpxbAdamw a, const double* partial, long long partials) {
  waitForPrevious();
  letNextStart();
  auto* s = static_cast<Scratch*>(a.scratch);
  if (l.first == 0) {
    float norm = 0.f;
    if (partial) norm = rootOfSum(partial, partials);
    else if (a.grad_norm) norm = *a.grad_norm;
    if (threadIdx.x == 0) {
      if (partial) *a.grad_norm = norm;
      float coef = 1.f;
      if (a.grad_norm) {
        const float c = a.max_norm / (norm + 1e-6f);
        coef = c < 1.f || c != c ? c : 1.f;
      }
      s->coef = coef;
    }
  }
  for (int i = threadIdx.x; i < l.count; i += blockDim.x) {
    const int t = ++*l.t[i].step;
    s->rates[l.first + i].stepSize = float(a.lr / (1.0 - pow(a.beta1, t)));
    s->rates[l.first + i].rootCorrection = float(1.0 / sqrt(1.0 - pow(a.beta2, t)));
  }
}

// Two elements.  m and v are taken in the formula's order, every product and sum rounded by
// itself: 8-bit codes then fall as those of any plain 32-bit computation do.  The root and the
// quotient are the approximate ones (2 units in the last place of 32 bits): they touch the weight's
// own step, and the exact ones would make the 8-bit kernel wait for arithmetic.  The fastest ones also
// take a v under 2^-126 for zero.  Next to an `eps` of 2^-39 or more times the root's correction a root
// under 2^-63 is nothing.  Under that (`eps` zero, or far below the usual ones) it may be all of the
// denominator, and a denominator's reciprocal may leave the range, as it does for a huge `eps`: kernels
// of their own (kWide) take roots of any v, and quotients.  (Both forms in one kernel: 1176 us instead of
// 1161 us for 323 M weights with clipping.)
template <bool kAll> __device__ __forceinline__ float2 roots(float2 v) {
  float2 r;
  if constexpr (kAll) {
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  } else {
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  }
  return r;
}
constexpr float kLeastNormal = 0x1p-126f;

struct Step {
  float beta1, beta2, rest1, rest2, eps, keep, stepSize, rootCorrection, coef;
  __device__ __forceinline__ void moments(float2 g, float2& m, float2& v) const {
    g = mul2(g, {coef, coef});
    // sums one by one: a packed sum would be contracted with its product, which rounds otherwise
    const float2 m1 = mul2(m, {beta1, beta1}), m2 = mul2(g, {rest1, rest1});
    m = {__fadd_rn(m1.x, m2.x), __fadd_rn(m1.y, m2.y)};
    const float2 v1 = mul2(v, {beta2, beta2}), v2 = mul2(mul2(g, {rest2, rest2}), g);
    v = {__fadd_rn(v1.x, v2.x), __fadd_rn(v1.y, v2.y)};
  }
  template <bool kWide> __device__ __forceinline__ void weights(float2& p, float2 m, float2 root) const {
    float2 below = fma2(root, {rootCorrection, rootCorrection}, {eps, eps});
    const float2 move = mul2(m, {-stepSize, -stepSize});
    if constexpr (kWide) {
      p = fma2(p, {keep, keep}, {__fdiv_rn(move.x, below.x), __fdiv_rn(move.y, below.y)});
    } else {
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(below.x) : "f"(below.x));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(below.y) : "f"(below.y));
      p = fma2(p, {keep, keep}, mul2(move, below));
    }
  }
  template <bool kWide> __device__ __forceinline__ void pair(float2& p, float2 g, float2& m, float2& v) const {
    moments(g, m, v);
    weights<kWide>(p, m, roots<kWide>(v));
  }
};

struct alignas(8) Codes { __nv_fp8x2_storage_t c[4]; };
__device__ __forceinline__ void decode(const Codes& x, float scale, float2 (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) f[i] = mul2(__half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(x.c[i], __NV_E4M3))), {scale, scale});
}
__device__ __forceinline__ Codes encode(const float2 (&f)[4]) {
  Codes x;
#pragma unroll
  for (int i = 0; i < 4; i++) x.c[i] = __nv_cvt_float2_to_fp8x2(f[i], __NV_SATFINITE, __NV_E4M3);
  return x;
}

// Eight elements from `at` on: a vector, or those below `end` one by one.
template <bool kVector, class V, class T> __device__ __forceinline__ V get(const T* p, long long at, long long end) {
  if constexpr (kVector) return *reinterpret_cast<const V*>(p + at);
  V x = {};
  T* e = reinterpret_cast<T*>(&x);
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (at + i < end) e[i] = p[at + i];
  return x;
}
template <bool kVector, class V, class T> __device__ __forceinline__ void put(T* p, long long at, long long end, const V& x) {
  if constexpr (kVector) {
    *reinterpret_cast<V*>(p + at) = x;
  } else {
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (at + i < end) p[at + i] = e[i];
  }
}

template <class T> __device__ __forceinline__ bool aligned(const T* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// 32-bit states, whole vectors: a thread has two runs of eight elements in flight, 96 bytes each.
template <class T, bool kWide> __device__ __forceinline__ void stepVectors(const tcpxbAdamwTensor& t, const Step& step, long long begin, long long end) {
  T* p = static_cast<T*>(t.p);
  const T* g = static_cast<const T*>(t.g);
  float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
#pragma unroll 2
  for (long long e = begin + threadIdx.x * 8; e < end; e += kThreads * 8) {
    float2 pp[4], gg[4], mm[4], vv[4];
    if (t.master) pairs(*reinterpret_cast<const Vec8<float>*>(t.master + e), pp);
    else pairs(*reinterpret_cast<const Vec8<T>*>(p + e), pp);
    pairs(*reinterpret_cast<const Vec8<T>*>(g + e), gg);
    pairs(*reinterpret_cast<const Vec8<float>*>(m + e), mm);
    pairs(*reinterpret_cast<const Vec8<float>*>(v + e), vv);
#pragma unroll
    for (int i = 0; i < 4; i++) step.pair<kWide>(pp[i], gg[i], mm[i], vv[i]);
    *reinterpret_cast<Vec8<float>*>(m + e) = rounded<float>(mm);
    *reinterpret_cast<Vec8<float>*>(v + e) = rounded<float>(vv);
    *reinterpret_cast<Vec8<T>*>(p + e) = rounded<T>(pp);
    if (t.master) *reinterpret_cast<Vec8<float>*>(t.master + e) = rounded<float>(pp);
  }
}

// 32-bit states, any alignment and the ends: one element a lane, four in flight.
template <class T, bool kWide> __device__ __forceinline__ void stepElements(const tcpxbAdamwTensor& t, const Step& step, long long begin, long long end) {
  T* p = static_cast<T*>(t.p);
  const T* g = static_cast<const T*>(t.g);
  float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
  for (long long e0 = begin + threadIdx.x; e0 < end; e0 += kThreads * 4) {
    float pp[4] = {}, gg[4] = {}, mm[4] = {}, vv[4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const long long e = e0 + i * kThreads;
      if (e < end) pp[i] = t.master ? t.master[e] : toFloat(p[e]), gg[i] = toFloat(g[e]), mm[i] = m[e], vv[i] = v[e];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      float2 w = {pp[i], pp[i + 1]}, m2 = {mm[i], mm[i + 1]}, v2 = {vv[i], vv[i + 1]};
      step.pair<kWide>(w, {gg[i], gg[i + 1]}, m2, v2);
      pp[i] = w.x, pp[i + 1] = w.y, mm[i] = m2.x, mm[i + 1] = m2.y, vv[i] = v2.x, vv[i + 1] = v2.y;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const long long e = e0 + i * kThreads;
      if (e >= end) break;
      m[e] = mm[i], v[e] = vv[i], p[e] = fromFloat<T>(pp[i]);
      if (t.master) t.master[e] = pp[i];
    }
  }
}

// 8-bit states: what a lane holds of a block.  W: the type that the weights are read in.
template <class T, class W> struct Raw {
  Vec8<W> w;
  Vec8<T> g;
  Codes m, v;
};
// Largest magnitude of the warp; NaN is left out (its code is NaN by itself).
__device__ __forceinline__ float warpTop(float x) {
  float y;
  asm("redux.sync.max.abs.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// About 320 instructions a block, of which 64 are the step itself: at this count issue and memory
// take about the same time, so the rest is kept short (the warp's maximum is one instruction, the four
// factors of a block are taken by four lanes at once).
template <bool kVector, bool kWide, class T, class W>
__device__ __forceinline__ void stepBlock(const Raw<T, W>& r, const tcpxbAdamwTensor& t, const Step& step, long long b, long long end, float& mScale, float& vScale) {
  const int lane = threadIdx.x % 32;
  const long long e = b + lane * 8;
  float2 pp[4], gg[4], mm[4], root[4];  // `root`: v until its root is taken
  pairs(r.w, pp);
  pairs(r.g, gg);
  decode(r.m, mScale, mm);
  decode(r.v, vScale, root);
  float topM = 0.f, topV = 0.f, least = INFINITY;
  // past the end everything is zero and stays so
#pragma unroll
  for (int i = 0; i < 4; i++) {
    root[i] = mul2(root[i], root[i]);
    step.moments(gg[i], mm[i], root[i]);
    least = min3(least, root[i].x, root[i].y);
  }
  if (kWide || least < kLeastNormal) {
    // the root is a state, which no `eps` hides
#pragma unroll
    for (int i = 0; i < 4; i++) root[i] = roots<true>(root[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) root[i] = roots<false>(root[i]);
  }
  least = INFINITY;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    step.weights<kWide>(pp[i], mm[i], root[i]);
    topM = max3(topM, fabsf(mm[i].x), fabsf(mm[i].y));
    topV = max3(topV, root[i].x, root[i].y);
    least = min3(least, root[i].x, root[i].y);
  }
  put<kVector>(static_cast<T*>(t.p), e, end, rounded<T>(pp));
  if constexpr (!std::is_same_v<T, W>) put<kVector>(t.master, e, end, rounded<float>(pp));
  topM = warpTop(topM), topV = warpTop(topV);
  // lanes 0 and 1 take the factors to codes, 2 and 3 the scales, of m and of the root.  Below 1e-30
  // a block is held as zeros: the factor would leave the range.
  const float top = lane & 1 ? topV : topM;
  float ratio = lane & 2 ? top * (1.f / kE4m3Max) : kE4m3Max * __frcp_rn(top);
  if (!(top >= 1e-30f)) ratio = 0.f;
  const float toM = __shfl_sync(0xffffffffu, ratio, 0), toV = __shfl_sync(0xffffffffu, ratio, 1);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    mm[i] = mul2(mm[i], {toM, toM});
    root[i] = mul2(root[i], {toV, toV});
  }
  if (least * toV < kLeastCode) {
    // rare: roots under the smallest code above zero become that code, zeros stay
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (root[i].x > 0.f) root[i].x = fmaxf(root[i].x, kLeastCode);
      if (root[i].y > 0.f) root[i].y = fmaxf(root[i].y, kLeastCode);
    }
  }
  put<kVector>(static_cast<__nv_fp8_storage_t*>(t.m), e, end, encode(mm));
  put<kVector>(static_cast<__nv_fp8_storage_t*>(t.v), e, end, encode(root));
  mScale = __shfl_sync(0xffffffffu, ratio, 2), vScale = __shfl_sync(0xffffffffu, ratio, 3);
}

template <int kBytes> __device__ __forceinline__ void copyAsync(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "n"(kBytes) : "memory");
}

// The blocks of a chunk, every fourth one by a warp.  A lane copies its own share of the blocks
// ahead into shared memory, three of them in flight (a register prefetch of one left memory idle:
// 0.66 ms for 323 M weights with no arithmetic at all).  The chunk's scales are read before the
// first block and written after the last: one in between waits for the stores to its neighbours
// (0.94 ms).
constexpr int kSmallWarps = 4, kStages = 4;
static_assert(kChunk / TCPXB_ADAMW_BLOCK / kSmallWarps <= 32, "a lane holds the scales of one block of its warp");

template <class T, class W, bool kWide> __device__ __forceinline__ void stepBlocks(char* shared, const tcpxbAdamwTensor& t, const Step& step, long long begin, long long end, bool vectors) {
  using Share = Raw<T, W>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Share* ring = reinterpret_cast<Share*>(shared) + warp * kStages * 32 + lane;  // kStages apart by 32
  const W* weights = static_cast<const W*>(std::is_same_v<T, W> ? t.p : t.master);
  const int blocks = int((end - begin + TCPXB_ADAMW_BLOCK - 1) / TCPXB_ADAMW_BLOCK), whole = vectors ? int((end - begin) / TCPXB_ADAMW_BLOCK) : 0;
  const long long block0 = begin / TCPXB_ADAMW_BLOCK;
  float mScale = 0.f, vScale = 0.f;  // of the warp's block number `lane`
  if (warp + kSmallWarps * lane < blocks) {
    mScale = t.m_scale[block0 + warp + kSmallWarps * lane];
    vScale = t.v_scale[block0 + warp + kSmallWarps * lane];
  }
  const auto copy = [&](int k) {
    const int n = warp + kSmallWarps * k;
    if (n < whole) {
      const long long e = begin + n * TCPXB_ADAMW_BLOCK + lane * 8;
      Share* to = ring + k % kStages * 32;
#pragma unroll
      for (int i = 0; i < int(sizeof(Vec8<W>)); i += 16) copyAsync<16>(reinterpret_cast<char*>(&to->w) + i, reinterpret_cast<const char*>(weights + e) + i);
#pragma unroll
      for (int i = 0; i < int(sizeof(Vec8<T>)); i += 16)
        copyAsync<16>(reinterpret_cast<char*>(&to->g) + i, reinterpret_cast<const char*>(static_cast<const T*>(t.g) + e) + i);
      copyAsync<8>(&to->m, static_cast<const char*>(t.m) + e);
      copyAsync<8>(&to->v, static_cast<const char*>(t.v) + e);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; k++) copy(k);
  int k = 0;
#pragma unroll 1
  for (; warp + kSmallWarps * k < whole; k++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    const Share r = ring[k % kStages * 32];  // a lane reads what it copied itself
    copy(k + kStages - 1);
    float m = __shfl_sync(0xffffffffu, mScale, k), v = __shfl_sync(0xffffffffu, vScale, k);
    stepBlock<true, kWide>(r, t, step, begin + (warp + kSmallWarps * k) * TCPXB_ADAMW_BLOCK, end, m, v);
    if (lane == k) mScale = m, vScale = v;
  }
#pragma unroll 1
  for (; warp + kSmallWarps * k < blocks; k++) {
    const long long b = begin + (warp + kSmallWarps * k) * TCPXB_ADAMW_BLOCK, e = b + lane * 8;
    const Share r = {get<false, Vec8<W>>(weights, e, end), get<false, Vec8<T>>(static_cast<const T*>(t.g), e, end),
                     get<false, Codes>(static_cast<const __nv_fp8_storage_t*>(t.m), e, end), get<false, Codes>(static_cast<const __nv_fp8_storage_t*>(t.v), e, end)};
    float m = __shfl_sync(0xffffffffu, mScale, k), v = __shfl_sync(0xffffffffu, vScale, k);
    stepBlock<false, kWide>(r, t, step, b, end, m, v);
    if (lane == k) mScale = m, vScale = v;
  }
  if (warp + kSmallWarps * lane < blocks) {
    t.m_scale[block0 + warp + kSmallWarps * lane] = mScale;
    t.v_scale[block0 + warp + kSmallWarps * lane] = vScale;
  }
}

// What a CTA works on: elements [begin, end) of a tensor.  The step goes through the list backwards: the
// gradients that the norm has read last are still in the L2.
template <class L> struct Chunk {
  int tensor;
  long long begin, end;
  __device__ __forceinline__ Chunk(const L& l, unsigned chunk) {
    tensor = tensorOf(l, chunk);
    begin = (long long)(chunk - (tensor ? l.end[tensor - 1] : 0)) * kChunk;
    end = min((long long)l.t[tensor].n, begin + kChunk);
  }
};
__device__ __forceinline__ Step stepOf(const tcpxbAdamw& a, int tensor) {
  const auto* s = static_cast<const Scratch*>(a.scratch);
  return {float(a.beta1), float(a.beta2), float(1 - a.beta1), float(1 - a.beta2), float(a.eps), float(1 - a.lr * a.weight_decay),
          s->rates[tensor].stepSize, s->rates[tensor].rootCorrection, s->coef};
}
__device__ __forceinline__ bool inVectors(const tcpxbAdamwTensor& t) { return aligned(t.p) && aligned(t.g) && aligned(t.m) && aligned(t.v) && aligned(t.master); }

template <class T, bool kWide, class L> __global__ void __launch_bounds__(kThreads, 4) stepKernel(const __grid_constant__ L l, const tcpxbAdamw a) {
  waitForPrevious();
  const Chunk<L> c(l, gridDim.x - 1 - blockIdx.x);
  const tcpxbAdamwTensor t = l.t[c.tensor];
  const Step step = stepOf(a, l.first + c.tensor);
  const long long whole = inVectors(t) ? c.begin + (c.end - c.begin) / 8 * 8 : c.begin;
  stepVectors<T, kWide>(t, step, c.begin, whole);
  stepElements<T, kWide>(t, step, whole, c.end);
}

template <class T, class W, bool kWide, class L> __global__ void __launch_bounds__(kSmallWarps * 32, sizeof(W) == 2 ? 8 : 4) stepSmallKernel(const __grid_constant__ L l, const tcpxbAdamw a) {
  waitForPrevious();
  __shared__ alignas(16) char shared[kSmallWarps * kStages * 32 * sizeof(Raw<T, W>)];
  const Chunk<L> c(l, gridDim.x - 1 - blockIdx.x);
  const tcpxbAdamwTensor t = l.t[c.tensor];
  const Step step = stepOf(a, l.first + c.tensor);
  stepBlocks<T, W, kWide>(shared, t, step, c.begin, c.end, inVectors(t));
}

template <class T, class L> __global__ void __launch_bounds__(kThreads) squaresKernel(const __grid_constant__ L l, double* partial) {
  letNextStart();
  const Chunk<L> c(l, blockIdx.x);
  const long long begin = c.begin, end = c.end;
  const T* g = static_cast<const T*>(l.t[c.tensor].g);
  // eight squares in 32 bits, those sums in 64: what rounding is left averages out
  double sum = 0;
  const long long whole = aligned(g) ? begin + (end - begin) / 8 * 8 : begin;
#pragma unroll 1
  for (long long e0 = begin + threadIdx.x * 8; e0 < whole; e0 += kThreads * 32) {
    Vec8<T> raw[4] = {};
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (e0 + u * kThreads * 8 < whole) raw[u] = *reinterpret_cast<const Vec8<T>*>(g + e0 + u * kThreads * 8);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      float2 x[4], y = {0.f, 0.f};
      pairs(raw[u], x);
#pragma unroll
      for (int k = 0; k < 4; k++) y = fma2(x[k], x[k], y);
      sum += y.x + y.y;
    }
  }
#pragma unroll 1
  for (long long e0 = whole + threadIdx.x; e0 < end; e0 += kThreads * 8) {
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const long long e = e0 + k * kThreads;
      const float x = e < end ? toFloat(g[e]) : 0.f;
      y += x * x;
    }
    sum += y;
  }
  const double all = blockSum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = all;
}

__global__ void __launch_bounds__(1024) normKernel(const double* partial, long long n, float* norm) {
  waitForPrevious();
  const float x = rootOfSum(partial, n);
  if (threadIdx.x == 0) *norm = x;
}

long long chunksOf(const tcpxbAdamwTensor& t) { return (t.n + kChunk - 1) / kChunk; }
size_t ratesBytes(int count) { return sizeof(Scratch) + sizeof(Rates) * size_t(count); }
size_t partialBytes(const tcpxbAdamwTensor* tensors, int count) {
  long long chunks = 0;
  for (int i = 0; tensors && i < count; i++) chunks += chunksOf(tensors[i]);
  return sizeof(double) * size_t(chunks + 1);
}

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

// Whether the first tensor with elements has 32-bit weights behind it.
bool withMasters(const tcpxbAdamwTensor* t, int count) {
  int i = 0;
  while (i < count && !t[i].n) i++;
  return i < count && t[i].master;
}

int check(const tcpxbAdamwTensor* t, int count, int dtype, bool step, int bits) {
  if (count < 0 || (count && !t)) return fail(TCPXB_T_INVALID, "null list");
  if (dtype != TCPXB_T_BF16 && dtype != TCPXB_T_F16 && dtype != TCPXB_T_F32) return fail(TCPXB_T_INVALID, "unknown type %d", dtype);
  const bool masters = withMasters(t, count);
  for (int i = 0; i < count; i++) {
    if (t[i].n < 0 || t[i].n > (1ll << 43)) return fail(TCPXB_T_INVALID, "tensor %d has a bad size", i);
    if (t[i].n && !t[i].g) return fail(TCPXB_T_INVALID, "tensor %d has no gradient", i);
    if (!step) continue;
    if (t[i].n && (bool(t[i].master) != masters || (t[i].master && dtype == TCPXB_T_F32)))
      return fail(TCPXB_T_INVALID, "32-bit masters stand behind all tensors or none, of a 16-bit type (tensor %d)", i);
    if (!t[i].step || (t[i].n && (!t[i].p || !t[i].m || !t[i].v || (bits == 8 && (!t[i].m_scale || !t[i].v_scale)))))
      return fail(TCPXB_T_INVALID, "tensor %d lacks its weights, states, scales or step", i);
  }
  return TCPXB_T_OK;
}

// Sums of squares of all chunks into `partial`; their number in *done.
template <class T> int squares(const tcpxbAdamwTensor* tensors, int count, double* partial, long long* done, cudaStream_t s) {
  return inLists(tensors, count, [&](const auto& l, long long chunks) {
    using L = std::decay_t<decltype(l)>;
    if (!chunks) return int(TCPXB_T_OK);
    squaresKernel<T, L><<<unsigned(chunks), kThreads, 0, s>>>(l, partial + *done);
    *done += chunks;
    return launched("gradient norm");
  });
}

template <class T, bool kWide> int step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw& a, cudaStream_t s) {
  const bool masters = withMasters(tensors, count);
  double* partial = nullptr;
  long long partials = 0;
  if (a.compute_norm) {
    partial = reinterpret_cast<double*>(static_cast<char*>(a.scratch) + ratesBytes(count));
    if (const int rc = squares<T>(tensors, count, partial, &partials, s)) return rc;
  }
  return inLists(tensors, count, [&](const auto& l, long long chunks) {
    using L = std::decay_t<decltype(l)>;
    const int threads = partials > 1024 ? 1024 : partials > 128 || l.count > 128 ? 384 : 128;
    if (const int rc = launchBehind(partials || l.first, prepareKernel<L>, 1, threads, 0, s, "adamw, rates", l, a, static_cast<const double*>(partial), partials)) return rc;
    if (!chunks) return int(TCPXB_T_OK);
    if (a.state_bits == 32) return launchBehind(true, stepKernel<T, kWide, L>, unsigned(chunks), kThreads, 0, s, "adamw", l, a);
    return launchBehind(true, masters ? stepSmallKernel<T, float, kWide, L> : stepSmallKernel<T, T, kWide, L>, unsigned(chunks), kSmallWarps * 32, 0, s, "adamw", l, a);
  });
}

template <class T> int step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw& a, cudaStream_t s) {
  // the correction, 1 / sqrt(1 - b2^t), is largest in the first step; above 2^100 the reciprocal of `eps` would be flushed
  return a.eps >= 0x1p-39 / sqrt(1 - a.beta2) && a.eps <= 0x1p100 ? step<T, false>(tensors, count, a, s) : step<T, true>(tensors, count, a, s);
}

template <class T> int gradNorm(const tcpxbAdamwTensor* tensors, int count, float* out, double* partial, cudaStream_t s) {
  long long done = 0;
  if (const int rc = squares<T>(tensors, count, partial, &done, s)) return rc;
  return launchBehind(done > 0, normKernel, 1, 1024, 0, s, "gradient norm, sum", static_cast<const double*>(partial), done, out);
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" size_t tcpxb_adamw_scratch_bytes(const tcpxbAdamwTensor* tensors, int count) {
  return count > 0 ? ratesBytes(count) + partialBytes(tensors, count) : 0;
}

extern "C" int tcpxb_adamw_step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw* a, void* stream) {
  if (!a || !a->scratch || reinterpret_cast<uintptr_t>(a->scratch) % 8 || (a->compute_norm && !a->grad_norm))
    return fail(TCPXB_T_INVALID, "the arguments, the scratch or the norm are null");
  if (a->state_bits != 8 && a->state_bits != 32) return fail(TCPXB_T_INVALID, "states have 8 or 32 bits, not %d", a->state_bits);
  if (const int rc = check(tensors, count, a->dtype, true, a->state_bits)) return rc;
  if (const int rc = use(a->device)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == TCPXB_T_BF16) return step<__nv_bfloat16>(tensors, count, *a, s);
  if (a->dtype == TCPXB_T_F16) return step<__half>(tensors, count, *a, s);
  return step<float>(tensors, count, *a, s);
}

extern "C" size_t tcpxb_grad_norm_scratch_bytes(const tcpxbAdamwTensor* tensors, int count) { return partialBytes(tensors, count); }

extern "C" int tcpxb_grad_norm(const tcpxbAdamwTensor* tensors, int count, int dtype, int device, float* norm, void* scratch, void* stream) {
  if (!norm || !scratch) return fail(TCPXB_T_INVALID, "null argument");
  if (const int rc = check(tensors, count, dtype, false, 32)) return rc;
  if (const int rc = use(device)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  auto* partial = static_cast<double*>(scratch);
  if (dtype == TCPXB_T_BF16) return gradNorm<__nv_bfloat16>(tensors, count, norm, partial, s);
  if (dtype == TCPXB_T_F16) return gradNorm<__half>(tensors, count, norm, partial, s);
  return gradNorm<float>(tensors, count, norm, partial, s);
}
