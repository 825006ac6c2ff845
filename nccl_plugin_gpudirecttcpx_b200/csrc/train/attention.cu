// Attention over [batch, tokens, heads, head size], forward and backward.
//
//   s_ij = scale q_i . k_j        P_i = softmax over the keys that query i sees
//   out_i = sum_j P_ij v_j        lse_i = log sum_j exp(s_ij)
//   D_i = dout_i . out_i          dS_ij = P_ij (dout_i . v_j - D_i)
//   dq_i = scale sum_j dS_ij k_j  dk_j = scale sum_i dS_ij q_i   dv_j = sum_i P_ij dout_i
//
// The backward pass keeps no probabilities: it takes them from the scores and lse again.
// One warp per row: lanes hold the head's elements, the softmax runs over the keys in one pass
// with a running maximum and sum.  Every sum is taken by one warp in a fixed order.
#include "common.h"

namespace tcpxb_train {
namespace {

constexpr int kMaxD = 128;
constexpr int kPer = kMaxD / 32;
constexpr int kWarps = 4;

__device__ __forceinline__ float warpSum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <class T> __device__ __forceinline__ void loadRow(const T* p, int d, float (&f)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int c = i * 32 + (threadIdx.x & 31);
    f[i] = c < d ? toFloat(p[c]) : 0.f;
  }
}
template <class T> __device__ __forceinline__ void storeRow(T* p, int d, const float (&f)[kPer], float by) {
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int c = i * 32 + (threadIdx.x & 31);
    if (c < d) p[c] = fromFloat<T>(f[i] * by);
  }
}
__device__ __forceinline__ float dot(const float (&a)[kPer], const float (&b)[kPer]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; i++) s += a[i] * b[i];
  return warpSum(s);
}

template <class T> __device__ __forceinline__ const T* row(const tcpxbHeads& x, int b, int s, int h) {
  return static_cast<const T*>(x.ptr) + b * x.stride_b + s * x.stride_s + h * x.stride_h;
}
__device__ __forceinline__ int keysOf(const tcpxbAttention& a, int b) {
  return a.key_lengths ? min(max(a.key_lengths[b], 0), a.sk) : a.sk;
}

template <class T> __global__ void forwardKernel(const tcpxbAttention a) {
  const long long r = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (r >= (long long)a.b * a.heads * a.sq) return;
  const int i = int(r % a.sq), h = int(r / a.sq % a.heads), b = int(r / a.sq / a.heads), kv = h / (a.heads / a.kv_heads);
  int keys = keysOf(a, b);
  if (a.causal) keys = min(keys, i + a.sk - a.sq + 1);
  float q[kPer], o[kPer] = {}, x[kPer];
  loadRow(row<T>(a.q, b, i, h), a.d, q);
  float top = -INFINITY, sum = 0.f;
  for (int j = 0; j < keys; j++) {
    loadRow(row<T>(a.k, b, j, kv), a.d, x);
    const float s = dot(q, x) * a.scale;
    const float next = fmaxf(top, s), keep = expf(top - next), p = expf(s - next);
    top = next;
    sum = sum * keep + p;
    loadRow(row<T>(a.v, b, j, kv), a.d, x);
#pragma unroll
    for (int c = 0; c < kPer; c++) o[c] = o[c] * keep + p * x[c];
  }
  storeRow(static_cast<T*>(a.out) + (((long long)b * a.sq + i) * a.heads + h) * a.d, a.d, o, keys > 0 ? 1.f / sum : 0.f);
  if ((threadIdx.x & 31) == 0) a.lse[((long long)b * a.heads + h) * a.sq + i] = keys > 0 ? top + logf(sum) : -INFINITY;
}

// dq of one row, and D for the other kernel.
template <class T> __global__ void backwardQueryKernel(const tcpxbAttention a) {
  const long long r = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (r >= (long long)a.b * a.heads * a.sq) return;
  const int i = int(r % a.sq), h = int(r / a.sq % a.heads), b = int(r / a.sq / a.heads), kv = h / (a.heads / a.kv_heads);
  int keys = keysOf(a, b);
  if (a.causal) keys = min(keys, i + a.sk - a.sq + 1);
  const long long at = (((long long)b * a.sq + i) * a.heads + h) * a.d;
  float q[kPer], go[kPer], dq[kPer] = {}, x[kPer];
  loadRow(row<T>(a.q, b, i, h), a.d, q);
  loadRow(row<T>(a.dout, b, i, h), a.d, go);
  loadRow(static_cast<const T*>(a.out) + at, a.d, x);
  const long long stat = ((long long)b * a.heads + h) * a.sq + i;
  const float lse = a.lse[stat], delta = dot(go, x);
  if ((threadIdx.x & 31) == 0) a.delta[stat] = delta;
  for (int j = 0; j < keys; j++) {
    loadRow(row<T>(a.v, b, j, kv), a.d, x);
    const float dp = dot(go, x);
    loadRow(row<T>(a.k, b, j, kv), a.d, x);
    const float ds = expf(dot(q, x) * a.scale - lse) * (dp - delta);
#pragma unroll
    for (int c = 0; c < kPer; c++) dq[c] += ds * x[c];
  }
  storeRow(static_cast<T*>(a.dq) + at, a.d, dq, a.scale);
}

// dk and dv of one key, over all query heads of its group.
template <class T> __global__ void backwardKeyKernel(const tcpxbAttention a) {
  const long long r = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (r >= (long long)a.b * a.kv_heads * a.sk) return;
  const int j = int(r % a.sk), kv = int(r / a.sk % a.kv_heads), b = int(r / a.sk / a.kv_heads), group = a.heads / a.kv_heads;
  float k[kPer], v[kPer], dk[kPer] = {}, dv[kPer] = {}, x[kPer], go[kPer];
  loadRow(row<T>(a.k, b, j, kv), a.d, k);
  loadRow(row<T>(a.v, b, j, kv), a.d, v);
  const int first = a.causal ? max(0, j - (a.sk - a.sq)) : 0;
  for (int h = kv * group; h < (kv + 1) * group && j < keysOf(a, b); h++) {
    for (int i = first; i < a.sq; i++) {
      loadRow(row<T>(a.q, b, i, h), a.d, x);
      loadRow(row<T>(a.dout, b, i, h), a.d, go);
      const long long stat = ((long long)b * a.heads + h) * a.sq + i;
      const float p = expf(dot(x, k) * a.scale - a.lse[stat]), ds = p * (dot(go, v) - a.delta[stat]);
#pragma unroll
      for (int c = 0; c < kPer; c++) dk[c] += ds * x[c], dv[c] += p * go[c];
    }
  }
  const long long at = (((long long)b * a.sk + j) * a.kv_heads + kv) * a.d;
  storeRow(static_cast<T*>(a.dk) + at, a.d, dk, a.scale);
  storeRow(static_cast<T*>(a.dv) + at, a.d, dv, 1.f);
}

int check(const tcpxbAttention* a, bool backward) {
  if (!a) return fail(TCPXB_T_INVALID, "null argument");
  if (a->b < 0 || a->sq < 0 || a->sk < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->d < 8 || a->d > kMaxD || a->d % 8)
    return fail(TCPXB_T_INVALID, "bad shape: b %d sq %d sk %d heads %d/%d d %d", a->b, a->sq, a->sk, a->heads, a->kv_heads, a->d);
  if (a->dtype != TCPXB_T_BF16 && a->dtype != TCPXB_T_F16) return fail(TCPXB_T_INVALID, "attention takes bf16 and fp16, not type %d", a->dtype);
  if (!(a->scale > 0.f) || a->scale > 1e30f) return fail(TCPXB_T_INVALID, "scale has to be finite and above zero");
  const bool queries = (long long)a->b * a->sq > 0, keys = (long long)a->b * a->sk > 0;
  if (queries && (!headsOk(a->q, 2) || !a->out || !a->lse)) return fail(TCPXB_T_INVALID, "q, out or lse is null or off the 16-byte boundary");
  if (keys && (!headsOk(a->k, 2) || !headsOk(a->v, 2))) return fail(TCPXB_T_INVALID, "k or v is null or off the 16-byte boundary");
  if (backward && ((queries && (!headsOk(a->dout, 2) || !a->dq || !a->delta)) || (keys && (!a->dk || !a->dv))))
    return fail(TCPXB_T_INVALID, "dout, dq, dk, dv or delta is null or off the 16-byte boundary");
  return TCPXB_T_OK;
}

template <class T> int forward(const tcpxbAttention& a, cudaStream_t s) {
  const long long rows = (long long)a.b * a.heads * a.sq;
  if (rows == 0) return TCPXB_T_OK;
  forwardKernel<T><<<unsigned((rows + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(a);
  return launched("attention forward");
}

template <class T> int backward(const tcpxbAttention& a, cudaStream_t s) {
  const long long rows = (long long)a.b * a.heads * a.sq, keys = (long long)a.b * a.kv_heads * a.sk;
  if (rows) {
    backwardQueryKernel<T><<<unsigned((rows + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(a);
    if (const int rc = launched("attention backward, queries")) return rc;
  }
  if (keys) backwardKeyKernel<T><<<unsigned((keys + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(a);
  return launched("attention backward, keys");
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" int tcpxb_attention_forward(const tcpxbAttention* a, void* stream) {
  if (const int rc = check(a, false)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return a->dtype == TCPXB_T_BF16 ? forward<__nv_bfloat16>(*a, s) : forward<__half>(*a, s);
}

extern "C" int tcpxb_attention_backward(const tcpxbAttention* a, void* stream) {
  if (const int rc = check(a, true)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  return a->dtype == TCPXB_T_BF16 ? backward<__nv_bfloat16>(*a, s) : backward<__half>(*a, s);
}
