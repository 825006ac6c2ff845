// Norms of queries and keys per head, with the position rotation in the same pass.
//
//   forward   r = rsqrt(mean(x^2) + eps), n = x r w,  (y_2i, y_2i+1) = n turned by the token's angle
//   backward  dn = dy turned back,  dw = sum over rows of dn (x r),
//             dx = r (dn w - (x r) mean(dn w (x r)))
//
// Memory-bound: every element is read and written once.  A head's row is held by a group of
// lanes, eight elements each (16 bytes of a 16-bit type), so the norm's sum is a few shuffles
// and each lane owns whole pairs.  All sums are 32-bit; the result is rounded once.
#include "common.h"

namespace tcpxb_train {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 148 * 4;  // also the rows of the partial sums of dw
constexpr int kMaxD = 256;

struct Row {
  long long token;
  int head;
  bool isQ;
};

__device__ __forceinline__ Row rowOf(const tcpxbNormRope& a, long long r) {
  const int all = a.heads + a.kv_heads;
  Row x;
  x.token = r / all;
  x.head = int(r % all);
  x.isQ = x.head < a.heads;
  if (!x.isQ) x.head -= a.heads;
  return x;
}

template <class T> __device__ __forceinline__ const T* input(const tcpxbHeads& x, const tcpxbNormRope& a, const Row& r) {
  return static_cast<const T*>(x.ptr) + r.token / a.s * x.stride_b + r.token % a.s * x.stride_s + r.head * x.stride_h;
}
template <class T> __device__ __forceinline__ T* output(void* q, void* k, const tcpxbNormRope& a, const Row& r) {
  return r.isQ ? static_cast<T*>(q) + (r.token * a.heads + r.head) * a.d : static_cast<T*>(k) + (r.token * a.kv_heads + r.head) * a.d;
}

// Four angles of a lane's eight elements; a token outside the tables has none.
__device__ __forceinline__ void angles(const tcpxbNormRope& a, long long token, int col, float (&c)[4], float (&s)[4]) {
  const long long p = a.pos ? a.pos[token] : token % a.s;
  if (p < 0 || p >= a.positions) {
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = s[i] = NAN;
    return;
  }
  const long long at = p * (a.d / 2) + col / 2;
#pragma unroll
  for (int i = 0; i < 4; i++) c[i] = a.cos[at + i], s[i] = a.sin[at + i];
}

template <int G> __device__ __forceinline__ float groupSum(float x) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <class T, int G, bool kNorm> __global__ void __launch_bounds__(kThreads) forwardKernel(const tcpxbNormRope a) {
  const long long rows = (long long)a.b * a.s * (a.heads + a.kv_heads);
  const int lane = threadIdx.x % G, col = lane * 8;
  const bool on = col < a.d;
  float w[2][8] = {};
  if (kNorm && on) {
    load8(static_cast<const T*>(a.wq) + col, w[0]);
    load8(static_cast<const T*>(a.wk) + col, w[1]);
  }
  // the groups of a warp leave the loop together, so the shuffles are whole
  const int perWarp = 32 / G;
  const long long step = (long long)gridDim.x * (kThreads / G);
  for (long long base = (long long)blockIdx.x * (kThreads / G) + threadIdx.x / 32 * perWarp; base < rows; base += step) {
    const long long r = base + threadIdx.x % 32 / G;
    const bool live = r < rows && on;
    const Row at = rowOf(a, r);
    float x[8] = {}, c[4], s[4];
    if (live) load8(input<T>(at.isQ ? a.q : a.k, a, at) + col, x);
    if (kNorm) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) sq += x[i] * x[i];
      const float inv = rsqrtf(groupSum<G>(sq) / a.d + a.eps);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] *= inv * (at.isQ ? w[0][i] : w[1][i]);
    }
    if (!live) continue;
    angles(a, at.token, col, c, s);
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
      y[2 * i + 1] = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
    }
    store8(output<T>(a.q_out, a.k_out, a, at) + col, y);
  }
}

template <class T, int G, bool kNorm> __global__ void __launch_bounds__(kThreads) backwardKernel(const tcpxbNormRope a) {
  const long long rows = (long long)a.b * a.s * (a.heads + a.kv_heads);
  const int lane = threadIdx.x % G, col = lane * 8;
  const bool on = col < a.d;
  float w[2][8] = {}, dw[2][8] = {};
  if (kNorm && on) {
    load8(static_cast<const T*>(a.wq) + col, w[0]);
    load8(static_cast<const T*>(a.wk) + col, w[1]);
  }
  const int perWarp = 32 / G;
  const long long step = (long long)gridDim.x * (kThreads / G);
  for (long long base = (long long)blockIdx.x * (kThreads / G) + threadIdx.x / 32 * perWarp; base < rows; base += step) {
    const long long r = base + threadIdx.x % 32 / G;
    const bool live = r < rows && on;
    const Row at = rowOf(a, r);
    float dy[8] = {}, dn[8] = {}, x[8] = {}, c[4], s[4];
    if (live) {
      load8(input<T>(at.isQ ? a.dq_out : a.dk_out, a, at) + col, dy);
      if (kNorm) load8(input<T>(at.isQ ? a.q : a.k, a, at) + col, x);
      angles(a, at.token, col, c, s);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        dn[2 * i] = dy[2 * i] * c[i] + dy[2 * i + 1] * s[i];
        dn[2 * i + 1] = dy[2 * i + 1] * c[i] - dy[2 * i] * s[i];
      }
    }
    if (kNorm) {
      float sq = 0.f, mix = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        sq += x[i] * x[i];
        mix += dn[i] * (at.isQ ? w[0][i] : w[1][i]) * x[i];
      }
      const float inv = rsqrtf(groupSum<G>(sq) / a.d + a.eps);
      const float mean = groupSum<G>(mix) * inv / a.d;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float xh = x[i] * inv;
        if (at.isQ) dw[0][i] += dn[i] * xh;
        else dw[1][i] += dn[i] * xh;
        dn[i] = inv * (dn[i] * (at.isQ ? w[0][i] : w[1][i]) - xh * mean);
      }
    }
    if (live) store8(output<T>(a.dq, a.dk, a, at) + col, dn);
  }
  if (!kNorm) return;
  // the block's groups, one after another in a fixed order
  __shared__ float sums[2 * kMaxD];
  for (int g = 0; g < kThreads / G; g++) {
    if (threadIdx.x / G == g && on) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 8; i++) sums[t * kMaxD + col + i] = (g ? sums[t * kMaxD + col + i] : 0.f) + dw[t][i];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.d; i += kThreads)
    a.partial[(long long)blockIdx.x * 2 * a.d + i] = sums[i / a.d * kMaxD + i % a.d];
}

// dw: the blocks' partial sums, in the order of the blocks.
template <class T> __global__ void weightKernel(const tcpxbNormRope a, int blocks) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= 2 * a.d) return;
  float sum = 0.f;
  for (int b = 0; b < blocks; b++) sum += a.partial[(long long)b * 2 * a.d + i];
  static_cast<T*>(i < a.d ? a.dwq : a.dwk)[i % a.d] = fromFloat<T>(sum);
}

int check(const tcpxbNormRope* a, bool backward) {
  if (!a) return fail(TCPXB_T_INVALID, "null argument");
  if (a->dtype != TCPXB_T_BF16 && a->dtype != TCPXB_T_F16 && a->dtype != TCPXB_T_F32) return fail(TCPXB_T_INVALID, "unknown type %d", a->dtype);
  if (a->b < 0 || a->s < 0 || a->heads < 1 || a->kv_heads < 1 || a->d < 8 || a->d > kMaxD || a->d % 8)
    return fail(TCPXB_T_INVALID, "bad shape: b %d s %d heads %d/%d d %d", a->b, a->s, a->heads, a->kv_heads, a->d);
  if (!a->wq != !a->wk) return fail(TCPXB_T_INVALID, "weights for queries and keys come together");
  if ((long long)a->b * a->s == 0) return TCPXB_T_OK;
  const int es = a->dtype == TCPXB_T_F32 ? 4 : 2;
  if (!a->cos || !a->sin || (!a->pos && a->positions < a->s)) return fail(TCPXB_T_INVALID, "tables are missing or shorter than the sequence");
  const bool needX = !backward || a->wq;
  if (needX && (!headsOk(a->q, es) || !headsOk(a->k, es))) return fail(TCPXB_T_INVALID, "q or k is null or off the 16-byte boundary");
  if (!backward && (!a->q_out || !a->k_out)) return fail(TCPXB_T_INVALID, "an output is null");
  if (backward && (!headsOk(a->dq_out, es) || !headsOk(a->dk_out, es) || !a->dq || !a->dk || (a->wq && (!a->dwq || !a->dwk || !a->partial))))
    return fail(TCPXB_T_INVALID, "a gradient or the scratch is null or off the 16-byte boundary");
  return TCPXB_T_OK;
}

template <class T, int G> int run(const tcpxbNormRope& a, bool backward, cudaStream_t s) {
  const long long rows = (long long)a.b * a.s * (a.heads + a.kv_heads), perBlock = kThreads / G;
  const int blocks = int(rows < kMaxBlocks * perBlock ? (rows + perBlock - 1) / perBlock : kMaxBlocks);
  if (!backward) {
    if (!blocks) return TCPXB_T_OK;
    if (a.wq) forwardKernel<T, G, true><<<blocks, kThreads, 0, s>>>(a);
    else forwardKernel<T, G, false><<<blocks, kThreads, 0, s>>>(a);
    return launched("norm and rotation, forward");
  }
  if (blocks) {
    if (a.wq) backwardKernel<T, G, true><<<blocks, kThreads, 0, s>>>(a);
    else backwardKernel<T, G, false><<<blocks, kThreads, 0, s>>>(a);
    if (const int rc = launched("norm and rotation, backward")) return rc;
  }
  if (a.wq) weightKernel<T><<<(2 * a.d + 63) / 64, 64, 0, s>>>(a, blocks);
  return launched("norm and rotation, weights");
}

template <class T> int byWidth(const tcpxbNormRope& a, bool backward, cudaStream_t s) {
  if (a.d <= 16) return run<T, 2>(a, backward, s);
  if (a.d <= 32) return run<T, 4>(a, backward, s);
  if (a.d <= 64) return run<T, 8>(a, backward, s);
  if (a.d <= 128) return run<T, 16>(a, backward, s);
  return run<T, 32>(a, backward, s);
}

int dispatch(const tcpxbNormRope* a, bool backward, void* stream) {
  if (const int rc = check(a, backward)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == TCPXB_T_BF16) return byWidth<__nv_bfloat16>(*a, backward, s);
  if (a->dtype == TCPXB_T_F16) return byWidth<__half>(*a, backward, s);
  return byWidth<float>(*a, backward, s);
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" size_t tcpxb_norm_rope_scratch_bytes(int d) { return d > 0 ? sizeof(float) * 2 * d * kMaxBlocks : 0; }
extern "C" int tcpxb_norm_rope_forward(const tcpxbNormRope* a, void* stream) { return dispatch(a, false, stream); }
extern "C" int tcpxb_norm_rope_backward(const tcpxbNormRope* a, void* stream) { return dispatch(a, true, stream); }
