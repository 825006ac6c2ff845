// Norms of queries and keys per head, with the position rotation in the same pass.
//
//   forward   r = rsqrt(mean(x^2) + eps), n = x r w,  (y_2i, y_2i+1) = n turned by the token's angle
//   backward  dn = dy turned back,  dw = sum over rows of dn (x r),
//             dx = r (dn w - (x r) mean(dn w (x r)))
//
// Memory-bound: every element is read and written once.  A head's row is held by a group of
// lanes, eight elements each (16 bytes of a 16-bit type), so the norm's sum is a few shuffles
// and each lane owns whole pairs.  A block works on queries or on keys, and a warp takes a few
// heads of one token at a time: their loads are all in flight before the first is used, and the
// token's angles and the weight are read once for them.  All sums are 32-bit; the result is
// rounded once.
#include "common.h"

namespace tcpxb_train {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxBlocks = 148 * 4;  // of the backward pass: the rows of the partial sums of dw
constexpr int kMaxD = 256;

// Rows that a lane group has in flight.
template <class T> constexpr int kRows = sizeof(T) == 2 ? 4 : 2;

// What a launch does to queries, and to keys.
struct Side {
  tcpxbHeads x, dy;
  const void* w;
  void* out;
  int heads;
  unsigned parts, units;  // warps' shares of a token, and of all tokens
};
struct Job {
  Side side[2];  // queries, keys
  const float *cos, *sin;
  const int64_t* pos;
  float* partial;
  unsigned s, qBlocks, kBlocks;
  int d, positions;
  float eps, perD;
};

// The token and the first of the heads that a warp does next.
struct Unit {
  unsigned token, batch, at;  // at: the token's number in its batch
  int head;
};
template <class T, int G> __device__ __forceinline__ Unit unitOf(const Job& j, const Side& side, unsigned u) {
  Unit x;
  x.token = u / side.parts;
  x.head = int(u - x.token * side.parts) * (32 / G * kRows<T>) + int(threadIdx.x % 32 / G);
  x.batch = x.token / j.s;
  x.at = x.token - x.batch * j.s;
  return x;
}
template <class T> __device__ __forceinline__ const T* input(const tcpxbHeads& x, const Unit& u, int col) {
  return static_cast<const T*>(x.ptr) + u.batch * x.stride_b + u.at * x.stride_s + u.head * x.stride_h + col;
}

// Four angles of a lane's eight elements; a token outside the tables has none.
__device__ __forceinline__ void angles(const Job& j, const Unit& u, int col, float (&c)[4], float (&s)[4]) {
  const long long p = j.pos ? j.pos[u.token] : u.at;
  if (p < 0 || p >= j.positions) {
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = s[i] = NAN;
    return;
  }
  const long long at = p * (j.d / 2) + col / 2;  // a multiple of four
  const float4 x = *reinterpret_cast<const float4*>(j.cos + at), y = *reinterpret_cast<const float4*>(j.sin + at);
  c[0] = x.x, c[1] = x.y, c[2] = x.z, c[3] = x.w;
  s[0] = y.x, s[1] = y.y, s[2] = y.z, s[3] = y.w;
}

template <int G> __device__ __forceinline__ float groupSum(float x) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <int G> __device__ __forceinline__ void groupSums(float& x, float& y) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    y += __shfl_xor_sync(0xffffffffu, y, o);
  }
}

template <class T> __device__ __forceinline__ void store(T* p, const float2 (&f)[4]) { *reinterpret_cast<Vec8<T>*>(p) = rounded<T>(f); }
__device__ __forceinline__ float sum(const float2 (&a)[4], const float2 (&b)[4]) {
  float2 s = mul2(a[0], b[0]);
#pragma unroll
  for (int i = 1; i < 4; i++) s = fma2(a[i], b[i], s);
  return s.x + s.y;
}

template <class T, int G, bool kNorm> __global__ void __launch_bounds__(kThreads) forwardKernel(const __grid_constant__ Job j) {
  const bool keys = blockIdx.x >= j.qBlocks;
  const Side& side = j.side[keys];
  const unsigned unit = (blockIdx.x - (keys ? j.qBlocks : 0)) * kWarps + threadIdx.x / 32;
  if (unit >= side.units) return;
  const int col = threadIdx.x % G * 8;
  const Unit u = unitOf<T, G>(j, side, unit);
  const bool on = col < j.d;
  const T* x = input<T>(side.x, u, col);
  T* y = static_cast<T*>(side.out) + ((long long)u.token * side.heads + u.head) * j.d + col;
  Vec8<T> raw[kRows<T>] = {};
#pragma unroll
  for (int i = 0; i < kRows<T>; i++)
    if (on && u.head + i * (32 / G) < side.heads) raw[i] = *reinterpret_cast<const Vec8<T>*>(x + i * (32 / G) * side.x.stride_h);
  float c[4] = {}, s[4] = {};
  float2 w[4] = {};
  if (on) {
    angles(j, u, col, c, s);
    if (kNorm) pairs(*reinterpret_cast<const Vec8<T>*>(static_cast<const T*>(side.w) + col), w);
  }
#pragma unroll
  for (int i = 0; i < kRows<T>; i++) {
    float2 f[4];
    pairs(raw[i], f);
    if (kNorm) {
      const float r = rsqrtf(groupSum<G>(sum(f, f)) * j.perD + j.eps);
#pragma unroll
      for (int k = 0; k < 4; k++) f[k] = mul2(mul2(f[k], {r, r}), w[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) f[k] = {f[k].x * c[k] - f[k].y * s[k], f[k].x * s[k] + f[k].y * c[k]};
    if (on && u.head + i * (32 / G) < side.heads) store(y + i * (32 / G) * j.d, f);
  }
}

// A few rows of a block's dw are in its lanes at the end: of queries in the first qBlocks, else of keys.
template <class T, int G, bool kNorm> __global__ void __launch_bounds__(kThreads, 2) backwardKernel(const __grid_constant__ Job j) {
  letNextStart();
  const bool keys = blockIdx.x >= j.qBlocks;
  const Side& side = j.side[keys];
  const unsigned block = blockIdx.x - (keys ? j.qBlocks : 0), blocks = keys ? j.kBlocks : j.qBlocks;
  const int col = threadIdx.x % G * 8;
  const bool on = col < j.d;
  float2 w[4] = {}, dw[4] = {};
  if (kNorm && on) pairs(*reinterpret_cast<const Vec8<T>*>(static_cast<const T*>(side.w) + col), w);
  for (unsigned unit = block * kWarps + threadIdx.x / 32; unit < side.units; unit += blocks * kWarps) {
    const Unit u = unitOf<T, G>(j, side, unit);
    const T *x = input<T>(side.x, u, col), *dy = input<T>(side.dy, u, col);
    T* dx = static_cast<T*>(side.out) + ((long long)u.token * side.heads + u.head) * j.d + col;
    Vec8<T> rawX[kRows<T>] = {}, rawY[kRows<T>] = {};
#pragma unroll
    for (int i = 0; i < kRows<T>; i++) {
      if (!on || u.head + i * (32 / G) >= side.heads) continue;
      rawY[i] = *reinterpret_cast<const Vec8<T>*>(dy + i * (32 / G) * side.dy.stride_h);
      if (kNorm) rawX[i] = *reinterpret_cast<const Vec8<T>*>(x + i * (32 / G) * side.x.stride_h);
    }
    float c[4] = {}, s[4] = {};
    if (on) angles(j, u, col, c, s);
#pragma unroll
    for (int i = 0; i < kRows<T>; i++) {
      const bool live = on && u.head + i * (32 / G) < side.heads;
      float2 f[4];
      pairs(rawY[i], f);
#pragma unroll
      for (int k = 0; k < 4; k++) f[k] = {f[k].x * c[k] + f[k].y * s[k], f[k].y * c[k] - f[k].x * s[k]};
      if (kNorm) {
        float2 x[4], g[4];
        pairs(rawX[i], x);
#pragma unroll
        for (int k = 0; k < 4; k++) g[k] = mul2(f[k], w[k]);
        // both sums go through the shuffles side by side: sum(g xh) = r sum(g x)
        float squares = sum(x, x), mix = sum(g, x);
        groupSums<G>(squares, mix);
        const float r = rsqrtf(squares * j.perD + j.eps), back = -r * r * (mix * j.perD) * r;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if (live) dw[k] = fma2(f[k], mul2(x[k], {r, r}), dw[k]);
          f[k] = fma2(x[k], {back, back}, mul2(g[k], {r, r}));
        }
      }
      if (live) store(dx + i * (32 / G) * j.d, f);
    }
  }
  if constexpr (kNorm) {
    // the groups of a warp by shuffles, then the block's warps, in a fixed order
    __shared__ float sums[kWarps][kMaxD];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      float x = k % 2 ? dw[k / 2].y : dw[k / 2].x;
#pragma unroll
      for (int o = 16; o; o >>= 1)
        if (o >= G) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (threadIdx.x % 32 < G && on) sums[threadIdx.x / 32][col + k] = x;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < j.d; i += kThreads) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; k++) x += sums[k][i];
      j.partial[(long long)blockIdx.x * j.d + i] = x;
    }
  }
}

// dw: the blocks' partial sums.  A block has 32 columns of one weight, and 32 warps that each take
// every 32nd row.
template <class T> __global__ void __launch_bounds__(1024) weightKernel(const __grid_constant__ Job j, T* dwq, T* dwk) {
  waitForPrevious();
  __shared__ float sums[32][33];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32, i = blockIdx.x * 32 + x;
  const unsigned first = blockIdx.y ? j.qBlocks : 0, end = blockIdx.y ? j.qBlocks + j.kBlocks : j.qBlocks;
  float part = 0.f;
  if (i < j.d) {
#pragma unroll 4
    for (unsigned b = first + y; b < end; b += 32) part += j.partial[(long long)b * j.d + i];
  }
  sums[y][x] = part;
  __syncthreads();
  // the sum of column y, taken by warp y
  part = sums[x][y];
#pragma unroll
  for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  const int c = blockIdx.x * 32 + y;
  if (x == 0 && c < j.d) (blockIdx.y ? dwk : dwq)[c] = fromFloat<T>(part);
}

int check(const tcpxbNormRope* a, bool backward) {
  if (!a) return fail(TCPXB_T_INVALID, "null argument");
  if (a->dtype != TCPXB_T_BF16 && a->dtype != TCPXB_T_F16 && a->dtype != TCPXB_T_F32) return fail(TCPXB_T_INVALID, "unknown type %d", a->dtype);
  if (a->b < 0 || a->s < 0 || a->heads < 1 || a->kv_heads < 1 || a->d < 8 || a->d > kMaxD || a->d % 8)
    return fail(TCPXB_T_INVALID, "bad shape: b %d s %d heads %d/%d d %d", a->b, a->s, a->heads, a->kv_heads, a->d);
  if ((long long)a->b * a->s * ((long long)a->heads + a->kv_heads) >= 1ll << 31)
    return fail(TCPXB_T_INVALID, "at most 2^31 - 1 rows: b %d s %d heads %d/%d", a->b, a->s, a->heads, a->kv_heads);
  if (!a->wq != !a->wk) return fail(TCPXB_T_INVALID, "weights for queries and keys come together");
  if (backward && a->wq && (!a->dwq || !a->dwk || !a->partial)) return fail(TCPXB_T_INVALID, "a weight's gradient or the scratch is null");
  if ((long long)a->b * a->s == 0) return TCPXB_T_OK;
  const int es = a->dtype == TCPXB_T_F32 ? 4 : 2;
  if (!a->cos || !a->sin || (!a->pos && a->positions < a->s)) return fail(TCPXB_T_INVALID, "tables are missing or shorter than the sequence");
  for (const void* p : {static_cast<const void*>(a->cos), static_cast<const void*>(a->sin), a->wq, a->wk})
    if (reinterpret_cast<uintptr_t>(p) % 16) return fail(TCPXB_T_INVALID, "a table or weight is off the 16-byte boundary");
  const bool needX = !backward || a->wq;
  if (needX && (!headsOk(a->q, es) || !headsOk(a->k, es))) return fail(TCPXB_T_INVALID, "q or k is null or off the 16-byte boundary");
  if (!backward && (!a->q_out || !a->k_out)) return fail(TCPXB_T_INVALID, "an output is null");
  if (backward && (!headsOk(a->dq_out, es) || !headsOk(a->dk_out, es) || !a->dq || !a->dk))
    return fail(TCPXB_T_INVALID, "a gradient is null or off the 16-byte boundary");
  return TCPXB_T_OK;
}

template <class T, int G> int run(const tcpxbNormRope& a, bool backward, cudaStream_t s) {
  const unsigned tokens = unsigned(a.b) * unsigned(a.s), perUnit = 32 / G * kRows<T>;
  const auto side = [&](const tcpxbHeads& x, const tcpxbHeads& dy, const void* w, void* out, int heads) {
    const unsigned parts = (unsigned(heads) + perUnit - 1) / perUnit;
    return Side{x, dy, w, out, heads, parts, tokens * parts};
  };
  Job j;
  j.side[0] = side(a.q, a.dq_out, a.wq, backward ? a.dq : a.q_out, a.heads);
  j.side[1] = side(a.k, a.dk_out, a.wk, backward ? a.dk : a.k_out, a.kv_heads);
  j.cos = a.cos, j.sin = a.sin, j.pos = a.pos, j.partial = a.partial;
  j.s = unsigned(a.s), j.d = a.d, j.positions = a.positions, j.eps = a.eps, j.perD = 1.f / float(a.d);
  j.qBlocks = (j.side[0].units + kWarps - 1) / kWarps, j.kBlocks = (j.side[1].units + kWarps - 1) / kWarps;
  if (!backward) {
    if (!tokens) return TCPXB_T_OK;
    if (a.wq) forwardKernel<T, G, true><<<j.qBlocks + j.kBlocks, kThreads, 0, s>>>(j);
    else forwardKernel<T, G, false><<<j.qBlocks + j.kBlocks, kThreads, 0, s>>>(j);
    return launched("norm and rotation, forward");
  }
  if (a.wq && j.qBlocks + j.kBlocks > unsigned(kMaxBlocks)) {
    // the partial sums' rows are given out by the two sides' work
    const unsigned long long all = (unsigned long long)j.qBlocks + j.kBlocks;
    unsigned k = unsigned(j.kBlocks * (unsigned long long)kMaxBlocks / all);
    k = k < 1 ? 1 : k > unsigned(kMaxBlocks) - 1 ? unsigned(kMaxBlocks) - 1 : k;
    j.kBlocks = k < j.kBlocks ? k : j.kBlocks;
    j.qBlocks = unsigned(kMaxBlocks) - k < j.qBlocks ? unsigned(kMaxBlocks) - k : j.qBlocks;
  }
  if (tokens) {
    if (a.wq) backwardKernel<T, G, true><<<j.qBlocks + j.kBlocks, kThreads, 0, s>>>(j);
    else backwardKernel<T, G, false><<<j.qBlocks + j.kBlocks, kThreads, 0, s>>>(j);
    if (const int rc = launched("norm and rotation, backward")) return rc;
  }
  if (!a.wq) return TCPXB_T_OK;
  return launchBehind(tokens > 0, weightKernel<T>, dim3((a.d + 31) / 32, 2), 1024, 0, s, "norm and rotation, weights", j, static_cast<T*>(a.dwq), static_cast<T*>(a.dwk));
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
  if (const int rc = use(a->device)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == TCPXB_T_BF16) return byWidth<__nv_bfloat16>(*a, backward, s);
  if (a->dtype == TCPXB_T_F16) return byWidth<__half>(*a, backward, s);
  return byWidth<float>(*a, backward, s);
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" size_t tcpxb_norm_rope_scratch_bytes(int d) { return d > 0 ? sizeof(float) * d * kMaxBlocks : 0; }
extern "C" int tcpxb_norm_rope_forward(const tcpxbNormRope* a, void* stream) { return dispatch(a, false, stream); }
extern "C" int tcpxb_norm_rope_backward(const tcpxbNormRope* a, void* stream) { return dispatch(a, true, stream); }
