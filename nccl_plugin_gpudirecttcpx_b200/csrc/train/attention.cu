// Attention over [batch, tokens, heads, head size], forward and backward.
//
//   s_ij = scale q_i . k_j        P_i = softmax over the keys that query i sees
//   out_i = sum_j P_ij v_j        lse_i = log sum_j exp(s_ij)
//   D_i = dout_i . out_i          dS_ij = P_ij (dout_i . v_j - D_i)
//   dq_i = scale sum_j dS_ij k_j  dk_j = scale sum_i dS_ij q_i   dv_j = sum_i P_ij dout_i
//
// The backward pass keeps no probabilities: it takes them from the scores and lse again.  It runs
// as two kernels, one that owns rows of dq and one that owns rows of dk and dv.  That costs seven
// matrix products where one kernel would need five, and in return no sum is ever taken by
// atomics: a gradient does not depend on the order in which blocks run, and no 32-bit copy of dq
// goes through memory.
//
// All three kernels work on tiles of scores, 128 rows high.  One warp loads tiles with TMA, one
// thread issues the matrix instructions, and eight warps turn scores into the operand of the
// next product, in tensor memory: the score tile is read into registers (forward a thread has a row, for
// the gradients of queries half of one, for those of keys two columns of every eight in four rows) and P or
// dS is written back over it in 16 bits.  A head size under 64 or between
// 64 and 128 fills its panel with zeros from the load.
//
// Head sizes above 64 take score tiles of 128 columns and one block on an SM: all of its tensor
// memory.  Up to 64 the products are half as long while the exponentials stay, so what counts is
// to keep the other units busy: tiles of 64 columns, half the tensor memory, two blocks on an SM
// that fill each other's waits, and each other's beginnings and ends.  Shared memory lets no more
// blocks onto an SM than its tensor memory serves, whichever of these kernels they are of, so an
// allocation never waits for a block of another cluster.
//
// A product that overwrites scores whose 16-bit form the product before it still reads is issued
// behind that one without a wait: the matrix instructions of a block run in the order of issue.
//
// Probabilities and score gradients are rounded to the inputs' type because the matrix units take
// operands of one type; sums, statistics and everything else are 32-bit.  In float16, whose range ends at
// 2^-24, the backward pass lifts both by powers of two and takes those out of the sums: see boundsKernel.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "tc.h"

namespace tcpxb_train {
namespace {

constexpr int kMaxD = 128;
constexpr int kTile = 128;
constexpr int kComputeWarps = 8, kLoadWarp = 8, kMmaWarp = 9;

// P: panels of 64 head elements.
template <int P> struct Tiling {
  static constexpr int kCols = P == 1 ? 64 : 128;  // of a score tile
  static constexpr int kHalf = kCols / 2;          // those of a thread in the backward pass
  static constexpr int kBlocks = P == 1 ? 2 : 1;   // on an SM
  static constexpr int kTmem = P == 1 ? 256 : 512;
  static constexpr int kHeadCols = P * 64;         // of a sum over scores
  static constexpr uint32_t kRowTile = P * kPanelBytes, kColTile = P * kCols * 128;
  // With one block the compute warps take registers from the others, for which two idle warps
  // complete a third warpgroup: 2 x 128 x 216 + 128 x 72 are the 384 x 168 of the launch.
  static constexpr int kThreads = P == 1 ? 320 : 384;
  static __device__ __forceinline__ void compute() {
    if constexpr (P == 2) moreRegisters<216>();
  }
  static __device__ __forceinline__ void other() {
    if constexpr (P == 2) fewerRegisters<72>();
  }
};
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Args {
  CUtensorMap q, k, v, dout;
  const void* out;
  const void *doutPtr, *vPtr;
  int64_t doutB, doutS, doutH, vB, vS, vH;
  const float2* bounds;
  int parts;
  void *o, *dq, *dk, *dv;
  float *lse, *delta;
  const int32_t* keyLengths;
  int32_t* status;
  int b, sq, sk, heads, kvHeads, d, causal;
  int split;  // blocks of a cluster that share a tile of keys
  float scale;
};

__device__ __forceinline__ int keysOf(const Args& a, int b) { return a.keyLengths ? min(max(a.keyLengths[b], 0), a.sk) : a.sk; }

// Keys that query i sees, of `keys`.
__device__ __forceinline__ int seenBy(const Args& a, int i, int keys) { return a.causal ? min(keys, max(0, i + a.sk - a.sq + 1)) : keys; }

template <int P> __device__ __forceinline__ int colTiles(int n) { return (n + Tiling<P>::kCols - 1) / Tiling<P>::kCols; }

// `R` rows in boxes of kCols.
template <int P, int R> __device__ __forceinline__ void loadTile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head, int batch) {
  constexpr int kBox = Tiling<P>::kCols;
#pragma unroll
  for (int p = 0; p < P; p++)
#pragma unroll
    for (int r = 0; r < R; r += kBox) tmaLoad(dst + p * R * 128 + r * 128, map, bar, p * 64, row + r, head, batch);
}

// Rows from `first` on become zero: what lies behind a key length may hold anything, and zero
// times NaN would reach the sums.  A warp does it between the load and the product that reads it.
template <int P> __device__ __forceinline__ void clearRows(uint32_t tile, int first) {
  constexpr int kCols = Tiling<P>::kCols;
  for (int r = first * 8 + int(threadIdx.x % 32); r < kCols * 8; r += 32) {
#pragma unroll
    for (int p = 0; p < P; p++)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + p * kCols * 128 + r * 16), "r"(0) : "memory");
  }
  fenceAsyncShared();
  __syncwarp();
}

struct Shared {
  uint64_t bars[32];
  uint32_t tmem;
  int dead[2];  // a wait has run out; the block has its tensor memory
  alignas(16) float stats[4][2][kTile];  // lse and D of a stage's queries
};
constexpr int kSharedBytes = 6144;
static_assert(sizeof(Shared) <= kSharedBytes, "barriers and statistics");

// Begins a block: the load warp has initialised the barriers and goes on to its loads, the others
// wait for that and for the tensor memory, and get its address.
template <int P> __device__ __forceinline__ uint32_t begin(int warp, uint32_t* tmem) {
  constexpr int kThreads = Tiling<P>::kThreads;
  if (warp == kLoadWarp) {
    asm volatile("bar.arrive 2, %0;" ::"n"(kThreads) : "memory");
    return 0;
  }
  if (warp == kMmaWarp) tmemAlloc(smemAddr(tmem), Tiling<P>::kTmem);
  tcBefore();
  asm volatile("bar.sync 2, %0;" ::"n"(kThreads) : "memory");
  tcAfter();
  return uniform(*tmem);
}

// A block where a wait ran out computes on memory that nothing has filled.  The flag is set before any of that can
// reach a sum, so the threads that store see it: their factors become NaN, and the outputs show it to a
// caller who has no status word.  A row that sees nothing is right all the same.
__device__ __forceinline__ float factor(bool sees, float by, volatile int* dead) { return !sees ? 0.f : *dead ? NAN : by; }
// Whether the status already tells of a wait that ran out: the block then does no work, so that a grid
// whose waits run out ends after the first of them, and what follows with the same status is void too.
__device__ __forceinline__ int isVoid(const int32_t* status) { return status && *reinterpret_cast<const volatile int32_t*>(status) == kStatusTimeout; }

template <int P> __device__ __forceinline__ void finish(const Args& a, uint32_t tmem, volatile int* dead) {
  tcBefore();
  __syncthreads();
  if (*dead) {
    // copies and products that nobody waited for may still be under way
    const uint64_t began = nowNs();
    while (nowNs() - began < 1000000) __nanosleep(1000);
    if (threadIdx.x == 0 && a.status) atomicMax(a.status, kStatusTimeout);
  }
  if (threadIdx.x / 32 == kMmaWarp) tmemFree(tmem, Tiling<P>::kTmem);
}

// Eight 32-bit values as 16 bytes; by zero they are zeros, whatever they were.
template <class T> __device__ __forceinline__ uint4 rounded8(const uint32_t* r, float by) {
  uint4 x = {};
  if (by != 0.f) {
    x.x = pack2<T>(__uint_as_float(r[0]) * by, __uint_as_float(r[1]) * by);
    x.y = pack2<T>(__uint_as_float(r[2]) * by, __uint_as_float(r[3]) * by);
    x.z = pack2<T>(__uint_as_float(r[4]) * by, __uint_as_float(r[5]) * by);
    x.w = pack2<T>(__uint_as_float(r[6]) * by, __uint_as_float(r[7]) * by);
  }
  return x;
}
// A warp's 32 accumulator rows, kCols of their columns from `begin` on, times each lane's `by`, to
// memory: row r goes to out + r * stride, where r < rows.  They are turned in `stage` (32 rows of
// kCols 16-bit elements, a tile that is no longer needed), so that a row's lanes write side by
// side; rows straight out of the lanes took 2000 to 4000 cycles of a block's end.
template <class T, int kCols>
__device__ __forceinline__ void storeRows(T* out, int64_t stride, int rows, uint32_t tmem, int begin, int d, float by, bool any, uint32_t stage) {
  constexpr int kChunks = kCols / 8;  // of 16 bytes in a row
  const int lane = threadIdx.x % 32;
  // the chunks of a row change places by its number: eight lanes never meet in a bank
  const auto place = [](int row, int c) { return uint32_t(row * kChunks + (c ^ (kChunks == 4 ? row / 2 % 4 : row % 8))) * 16; };
#pragma unroll
  for (int c = 0; c < kCols; c += 32) {
    uint32_t r[32] = {};
    if (any) {
      tmemLoad32(tmem + begin + c, r);
      tmemWaitLoad();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint4 x = rounded8<T>(r + i * 8, by);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + place(lane, c / 8 + i)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kChunks; i++) {
    const int row = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(stage + place(row, c)) : "memory");
    if (row < rows && begin + c * 8 < d) *reinterpret_cast<uint4*>(out + row * stride + begin + c * 8) = x;
  }
}

// A cluster of `split` blocks can share a tile of rows, each with a part of what the rows are summed
// over: at the end every block leaves its 32-bit sums in shared memory and adds up an equal part of
// the rows, always in the order of the blocks.
__device__ __forceinline__ void clusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Where 16-byte piece c of a row lies: pieces change places within 128 bytes, so that neither a
// column of rows nor the pieces of a row meet in a bank.
template <int kCols> __device__ __forceinline__ uint32_t pieceAt(uint32_t base, int row, int c) { return base + (row * (kCols / 4) + (c ^ row % 8)) * 16; }
// A value that block `rank` of the cluster has at `at` in its shared memory.
__device__ __forceinline__ float remote(uint32_t at, int rank) {
  float x;
  asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
// kPart columns of the thread's accumulator row into shared memory; NaN where a wait ran out.
template <int kCols, int kPart> __device__ __forceinline__ void leaveRow(uint32_t base, int row, uint32_t tmem, int begin, bool any, volatile int* dead) {
  const float nothing = uniform(*dead) ? NAN : 0.f;  // the loads want the whole warp
#pragma unroll
  for (int c = 0; c < kPart; c += 32) {
    uint32_t r[32];
    if (any && nothing == 0.f) {
      tmemLoad32(tmem + begin + c, r);
      tmemWaitLoad();
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) r[i] = __float_as_uint(nothing);
    }
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(pieceAt<kCols>(base, row, (begin + c + i) / 4)), "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]),
                   "r"(r[i + 3])
                   : "memory");
  }
}
// Adds eight elements of a row that block `rank` of the cluster has left, times `by`.
template <int kCols> __device__ __forceinline__ void addRow8(uint32_t base, int row, int c, int rank, float by, float (&sum)[8]) {
#pragma unroll
  for (int k = 0; k < 2; k++) {
    uint32_t at;
    float x[4];
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(pieceAt<kCols>(base, row, c * 2 + k)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(at) : "memory");
#pragma unroll
    for (int u = 0; u < 4; u++) sum[k * 4 + u] += x[u] * by;
  }
}

// ------------------------------------------------------------------ forward
// A block owns two tiles of queries; four warps do the softmax of each.  While one tile's scores
// are turned into probabilities, the matrix units work for the other one: out += P V of the
// last key tile, then the scores of the next.  A thread holds a whole row, so maximum and sum
// need no exchange.  The accumulator is rescaled only where a row's maximum has grown by more
// than 2^8 since its last rescaling: probabilities then reach 2^8, which costs no precision.
template <class T, int P> struct Forward {
  static constexpr int kSlots = P == 2 ? 4 : 8;  // tiles of keys and values in turn
  static constexpr uint32_t kTileBytes = Tiling<P>::kColTile, kQBytes = Tiling<P>::kRowTile;
  static constexpr size_t kShared = kSharedBytes + 1024 + 2 * kQBytes + kSlots * kTileBytes;
  static_assert(kSlots * kTileBytes >= 2 * kTile * Tiling<P>::kHeadCols * 4, "the sums of shared tiles fit the ring");
  enum { kQFull = 0, kFull = 2, kEmpty = kFull + kSlots, kSFull = kEmpty + kSlots, kPFull = kSFull + 2, kOFull = kPFull + 2, kBars = kOFull + 2 };
};

template <class T, int P, bool kSplit> __global__ void __launch_bounds__(Tiling<P>::kThreads, Tiling<P>::kBlocks) forwardKernel(const __grid_constant__ Args a) {
  using F = Forward<T, P>;
  using L = Tiling<P>;
  constexpr int kCols = L::kCols;
  static_assert(F::kBars <= 32, "barriers");
  extern __shared__ char raw[];
  const int split = kSplit ? a.split : 1;
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const uint32_t tile0 = (smemAddr(raw) + kSharedBytes + 1023) / 1024 * 1024, ring = tile0 + 2 * F::kQBytes;
  const auto bar = [&](int i) { return smemAddr(sh.bars) + 8 * i; };
  volatile int* dead = sh.dead;
  const int warp = uniform(int(threadIdx.x) / 32), lane = threadIdx.x % 32;
  // the longest blocks first, over all heads and batches: with a causal mask the last queries see the most keys
  const int q0 = (int(gridDim.z) - 1 - int(blockIdx.z)) * 2 * kTile, h = blockIdx.x / split, rank = blockIdx.x % split, b = blockIdx.y, kv = h / (a.heads / a.kvHeads);
  const int keys = keysOf(a, b);
  int all[2], n[2];  // tiles of keys that a tile of queries sees, and those of this block's part
#pragma unroll
  for (int t = 0; t < 2; t++) all[t] = q0 + t * kTile < a.sq ? colTiles<P>(seenBy(a, min(q0 + t * kTile + kTile, a.sq) - 1, keys)) : 0;
  const int every = max(all[0], all[1]), begun = int((long long)every * rank / split);

  const auto loadPair = [&](int i) {  // number i of K_0, V_0, K_1, ...
    const int slot = i % F::kSlots;
    barExpect(bar(F::kFull + slot), F::kTileBytes);
    loadTile<P, kCols>(ring + slot * F::kTileBytes, i & 1 ? &a.v : &a.k, bar(F::kFull + slot), (begun + i / 2) * kCols, kv, b);
  };
  if (warp == kLoadWarp) {
    if (lane == 0) {
      for (int i = 0; i < F::kBars; i++) barInit(bar(i), i >= F::kPFull && i < F::kOFull ? 4 : 1);
      dead[0] = isVoid(a.status), dead[1] = 0;
      fenceBarInit();
      fenceAsyncShared();
    }
    __syncwarp();
  }
  const uint32_t tmem = begin<P>(warp, &sh.tmem);
  if (warp == kMmaWarp) dead[1] = 1;
  const int most = uniform(*dead) ? 0 : int((long long)every * (rank + 1) / split) - begun;
#pragma unroll
  for (int t = 0; t < 2; t++) n[t] = min(max(all[t] - begun, 0), most);
  if (warp == kLoadWarp) {
    L::other();
    if (lane == 0) {
      for (int t = 0; t < 2; t++)
        if (n[t]) {
          barExpect(bar(F::kQFull + t), F::kQBytes);
          loadTile<P, kTile>(tile0 + t * F::kQBytes, &a.q, bar(F::kQFull + t), q0 + t * kTile, h, b);
          if (t == 0 || !n[0]) loadPair(0);
        }
      for (int i = 1; i < 2 * most; i++) {
        if (i >= F::kSlots) barWait(bar(F::kEmpty + i % F::kSlots), (i / F::kSlots - 1) & 1, dead);
        loadPair(i);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    L::other();
    const bool leader = electOne();
    const int steps = (a.d + 15) / 16;
    const uint32_t scores = mmaShape<T>(kCols, false), values = mmaShape<T>(steps * 16, true);
    for (int j = 0; j <= most; j++) {
      const int ik = 2 * j, iv = 2 * j - 1;  // numbers of K_j and V_j-1
      const uint32_t kTileAt = ring + ik % F::kSlots * F::kTileBytes, vTileAt = ring + (iv + F::kSlots) % F::kSlots * F::kTileBytes;
      if (j < most) barWait(bar(F::kFull + ik % F::kSlots), ik / F::kSlots & 1, dead);
      if (j) {
        barWait(bar(F::kFull + iv % F::kSlots), iv / F::kSlots & 1, dead);
        if ((begun + j) * kCols > keys && keys < a.sk) clearRows<P>(vTileAt, keys - (begun + j - 1) * kCols);
      }
      for (int t = 0; t < 2; t++) {
        const uint32_t s = tmem + t * kCols, o = tmem + 2 * kCols + t * L::kHeadCols;
        if (j && j <= n[t]) {
          barWait(bar(F::kPFull + t), (j - 1) & 1, dead);
          tcAfter();
          if (leader) {
            mmaTmemTile<kCols, kCols / 4>(o, s, vTileAt, values, j > 1);
            if (j == n[t]) mmaCommit(bar(F::kOFull + t));
          }
        }
        if (j < n[t]) {
          if (j == 0) barWait(bar(F::kQFull + t), 0, dead);
          if (leader) {
            // in issue order behind the product that reads P out of the same columns
            mmaTiles<P>(s, tile0 + t * F::kQBytes, kTileAt, scores, steps);
            mmaCommit(bar(F::kSFull + t));
          }
        }
      }
      if (leader) {
        // only where a load waits for it: no arrival may come after the block has gone
        if (ik + F::kSlots < 2 * most) mmaCommit(bar(F::kEmpty + ik % F::kSlots));
        if (j && iv + F::kSlots < 2 * most) mmaCommit(bar(F::kEmpty + iv % F::kSlots));
      }
      __syncwarp();
    }
  } else if (warp < kComputeWarps) {
    L::compute();
    const int t = warp / 4, row = warp % 4 * 32 + lane, i = q0 + t * kTile + row;
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const uint32_t s = tmem + t * kCols + lanes, o = tmem + 2 * kCols + t * L::kHeadCols + lanes;
    const float c = a.scale * kLog2e;
    const int seen = seenBy(a, i, keys);                       // of this row
    const int whole = seenBy(a, q0 + t * kTile, keys) / kCols;  // tiles that every row sees whole
    float top = -INFINITY;
    float2 sum2 = {0.f, 0.f};
    for (int j = 0; j < n[t]; j++) {
      barWait(bar(F::kSFull + t), j & 1, dead);
      tcAfter();
      uint32_t x[kCols];
      tmemLoad<kCols>(s, x);
      tmemWaitLoad();
      if (begun + j >= whole) {
        const int left = seen - (begun + j) * kCols;
#pragma unroll
        for (int k = 0; k < kCols; k++) x[k] = k < left ? x[k] : 0xff800000u;
      }
      float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < kCols; k += 8)
#pragma unroll
        for (int u = 0; u < 4; u++) m[u] = max3(m[u], __uint_as_float(x[k + u]), __uint_as_float(x[k + 4 + u]));
      const float now = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      const bool grown = (now - top) * c > 8.f || (top == -INFINITY && now > -INFINITY);
      if (__any_sync(0xffffffffu, grown)) {
        const float keep = grown ? exp2Fast((top - now) * c) : 1.f;
        if (grown) top = now;
        sum2 = mul2(sum2, {keep, keep});
        if (j) {
#pragma unroll 1
          for (int k = 0; k < a.d; k += 16) {
            uint32_t r[16];
            tmemLoad16(o + k, r);
            tmemWaitLoad();
#pragma unroll
            for (int u = 0; u < 16; u++) r[u] = __float_as_uint(__uint_as_float(r[u]) * keep);
            tmemStore16(o + k, r);
          }
        }
      }
      constexpr int kRun = P == 1 ? 32 : 64;  // columns that are stored at once
      const float base = top == -INFINITY ? 0.f : -top * c;
#pragma unroll
      for (int k = 0; k < kCols; k += kRun) {
        uint32_t p[kRun / 2];
#pragma unroll
        for (int u = 0; u < kRun; u += 2) {
          float2 e = fma2({__uint_as_float(x[k + u]), __uint_as_float(x[k + u + 1])}, {c, c}, {base, base});
          e.x = exp2Fast(e.x), e.y = exp2Fast(e.y);
          sum2 = add2(sum2, e);
          p[u / 2] = pack2<T>(e.x, e.y);
        }
        tmemStore<kRun / 2>(s + k / 2, p);
      }
      tmemWaitStore();
      tcBefore();
      __syncwarp();
      if (lane == 0) barArrive(bar(F::kPFull + t));
    }
    if (n[t]) {
      barWait(bar(F::kOFull + t), 0, dead);
      tcAfter();
    }
    const float sum = sum2.x + sum2.y;
    const bool live = i < a.sq;
    if constexpr (kSplit) {
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the other tile of queries reads the ring to its own end
      leaveRow<L::kHeadCols, L::kHeadCols>(ring + t * kTile * L::kHeadCols * 4, row, o, 0, n[t] > 0, dead);
      sh.stats[t][0][row] = top, sh.stats[t][1][row] = *dead ? NAN : sum;
    } else {
      // a row that sees nothing is zero, whatever its tile holds
      const float by = factor(seen > 0, 1.f / sum, dead);
      const int i0 = i - lane;  // the warp's first row
      storeRows<T, L::kHeadCols>(static_cast<T*>(a.o) + (((long long)b * a.sq + i0) * a.heads + h) * a.d, (int64_t)a.heads * a.d, a.sq - i0, o, 0, a.d, by,
                                 n[t] > 0, tile0 + t * F::kQBytes + warp % 4 * (F::kQBytes / 4));
      if (live) a.lse[((long long)b * a.heads + h) * a.sq + i] = seen > 0 ? by == by ? (top * c + log2f(sum)) * kLn2 : by : -INFINITY;
    }
  } else {
    L::other();
  }
  if constexpr (kSplit) {
    clusterSync();
    if (warp < kComputeWarps) {
      const float c = a.scale * kLog2e;
      const int rows = 2 * kTile / split, chunks = a.d / 8, count = rows * chunks;
      for (int k = threadIdx.x; k < count; k += kComputeWarps * 32) {
        const int r = rank * rows + k / chunks, t = r / kTile, row = r % kTile, chunk = k % chunks, i = q0 + r;
        // the blocks' sums are for maxima of their own
        float tops[8], sums[8], top = -INFINITY, sum = 0.f, o[8] = {};
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (u < split) {
            tops[u] = remote(smemAddr(&sh.stats[t][0][row]), u), sums[u] = remote(smemAddr(&sh.stats[t][1][row]), u);
            top = fmaxf(top, tops[u]);
          }
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (u < split && sums[u] != 0.f) {
            const float by = exp2Fast((tops[u] - top) * c);
            sum += sums[u] * by;
            addRow8<L::kHeadCols>(ring + t * kTile * L::kHeadCols * 4, row, chunk, u, by, o);
          }
        if (i >= a.sq) continue;
        const bool sees = seenBy(a, i, keys) > 0;
        *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (((long long)b * a.sq + i) * a.heads + h) * a.d + chunk * 8) =
            rounded8<T>(reinterpret_cast<const uint32_t*>(o), sees ? 1.f / sum : 0.f);
        if (chunk == 0) a.lse[((long long)b * a.heads + h) * a.sq + i] = sees ? (top * c + log2f(sum)) * kLn2 : -INFINITY;
      }
    }
    clusterSync();  // nobody leaves while its sums are read
  }
  finish<P>(a, tmem, dead);
}

// ------------------------------------------------------------------ backward, range of float16
// A probability among thousands of keys times a gradient of 1e-4 is under float16's smallest step, and
// dq and dk would be sums of zeros.  |dP_ij| and |D_i| are at most d max|dout| max|v| =: X, so the score
// gradients stay under 2.01 X: multiplied by 2^e with 2^13 <= 2^e X < 2^14 none of them overflows, and
// what still falls under the smallest step is 2^-38 of X.  It is exact and costs no instruction in the
// loops (a sum becomes a multiply-add).  Probabilities, at most one, are lifted by 2^14 for dv.
//
// The maxima are taken over each key head's group and batch, over the rows that see a key and the keys
// that can be seen; infinities and NaN are left out.  Up to kParts blocks share a key head's rows, about two
// blocks to an SM in all, and each leaves the maxima of its own; a kernel that needs them takes them of all.
// Memory-bound: every element of dout and v is read once, 14.8 us for 4 x 2048 tokens, 32/8 heads of 64 (42 MB; 17.6 us
// with a few blocks more than find room at once), of 480 us both ways.
constexpr int kParts = 32, kBoundsThreads = 1024;
constexpr float kProbabilityLift = 14.f, kProbabilityDrop = 0x1p-14f;  // the exponent, and what takes it out again

template <class T, int P> __global__ void __launch_bounds__(kBoundsThreads) boundsKernel(const __grid_constant__ Args a, float2* out) {
  letNextStart();
  constexpr int kWarps = kBoundsThreads / 32, kLanes = P * 8, kRows = kBoundsThreads / kLanes, kAhead = 4;
  const int kv = blockIdx.y, b = blockIdx.z, part = blockIdx.x, group = a.heads / a.kvHeads, keys = keysOf(a, b);
  const int col = int(threadIdx.x) % kLanes * 8;
  // of tokens [first, end): those of this part, all heads of a token side by side
  const auto most = [&](const T* x, int64_t token, int64_t head, int heads, int first, int end) {
    const int chunk = (end - first + a.parts - 1) / a.parts, begin = first + part * chunk;
    const int count = (min(begin + chunk, end) - begin) * heads;
    float top = 0.f;
    if (col >= a.d) return top;
    for (int i0 = int(threadIdx.x) / kLanes; i0 < count; i0 += kRows * kAhead) {
      Vec8<T> raw[kAhead] = {};
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int i = i0 + u * kRows;
        if (i < count) raw[u] = *reinterpret_cast<const Vec8<T>*>(x + (begin + i / heads) * token + i % heads * head + col);
      }
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        float2 f[4];
        pairs(raw[u], f);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float m = fabsf(f[k].x), n = fabsf(f[k].y);
          top = max3(top, m < INFINITY ? m : 0.f, n < INFINITY ? n : 0.f);
        }
      }
    }
    return top;
  };
  const int seeing = keys ? a.causal ? max(0, a.sq - a.sk) : 0 : a.sq;  // first query that sees a key
  const float g = most(static_cast<const T*>(a.doutPtr) + b * a.doutB + kv * group * a.doutH, a.doutS, a.doutH, group, seeing, a.sq);
  const float v = most(static_cast<const T*>(a.vPtr) + b * a.vB + kv * a.vH, a.vS, 0, 1, 0, keys);
  // values above zero are ordered as their bits are
  __shared__ unsigned tops[2][kWarps];
  const unsigned x = __reduce_max_sync(0xffffffffu, __float_as_uint(g)), y = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
  if (threadIdx.x % 32 == 0) tops[0][threadIdx.x / 32] = x, tops[1][threadIdx.x / 32] = y;
  __syncthreads();
  if (threadIdx.x < 32) {
    const unsigned m = __reduce_max_sync(0xffffffffu, tops[0][threadIdx.x]), n = __reduce_max_sync(0xffffffffu, tops[1][threadIdx.x]);
    if (threadIdx.x == 0) out[((long long)b * a.kvHeads + kv) * kParts + part] = {__uint_as_float(m), __uint_as_float(n)};
  }
}

template <class T> constexpr bool kLifted = std::is_same_v<T, __half>;
// 2^e, for a warp.
template <class T> __device__ __forceinline__ float liftOf(const Args& a, int b, int kv) {
  if (!kLifted<T> || !a.bounds) return 1.f;
  const int part = threadIdx.x % 32;
  const float2 top = part < a.parts ? a.bounds[((long long)b * a.kvHeads + kv) * kParts + part] : float2{};
  const unsigned x = __reduce_max_sync(0xffffffffu, __float_as_uint(top.x)), y = __reduce_max_sync(0xffffffffu, __float_as_uint(top.y));
  const unsigned all = __float_as_uint(__uint_as_float(x) * __uint_as_float(y) * float(a.d));  // 2^-45 to 2^39, or none
  return all ? __uint_as_float((127 + 13 + 127 - (all >> 23)) << 23) : 1.f;
}
// 1 / x of a power of two.
__device__ __forceinline__ float reciprocal(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }
// (y + minus) * lift, where `minus` has been lifted already.
template <class T> __device__ __forceinline__ float2 lifted(float2 y, float lift, float2 minus) {
  if constexpr (kLifted<T>) return fma2(y, {lift, lift}, minus);
  else return add2(y, minus);
}

// ------------------------------------------------------------------ backward, queries
// A block owns 128 queries and goes through the key tiles:  S = Q K^T, dP = dout V^T, then
// dq += dS K.  Two buffers of scores: the next tile's exponentials start while the matrix units
// still work on dP and dq of this one.  Both halves of the warps hold all rows, each half of the tile's keys.
// D_i is computed here and left for the other kernel: on the way in from dout and out; where all
// keys of the block lie in one tile, as sum_j P_ij dP_ij, which it equals.  In so short a row the
// rounding of out would be most of the gradients' error, and there the whole row is at hand.
template <class T, int P> struct Queries {
  static constexpr int kKSlots = P == 2 ? 3 : 5, kVSlots = P == 2 ? 2 : 3;
  static constexpr uint32_t kTileBytes = Tiling<P>::kColTile, kQBytes = Tiling<P>::kRowTile;
  static constexpr size_t kShared = 1024 + 1024 + 2 * kQBytes + (kKSlots + kVSlots) * kTileBytes;
  static_assert(kKSlots * kTileBytes >= kTile * Tiling<P>::kHeadCols * 4, "the sums of a shared tile fit the ring of keys");
  enum { kQFull = 0, kKFull = 1, kVFull = kKFull + kKSlots, kKEmpty = kVFull + kVSlots, kVEmpty = kKEmpty + kKSlots, kSFull = kVEmpty + kVSlots,
         kDpFull = kSFull + 2, kDsFull, kDone, kBars };
};

// A score that the row or key does not count for leaves exactly zero.
template <class T, int P, bool kSplit> __global__ void __launch_bounds__(Tiling<P>::kThreads, Tiling<P>::kBlocks) queryKernel(const __grid_constant__ Args a) {
  using F = Queries<T, P>;
  using L = Tiling<P>;
  constexpr int kCols = L::kCols, kHalf = L::kHalf;
  static_assert(F::kBars <= 32, "barriers");
  extern __shared__ char raw[];
  const int split = kSplit ? a.split : 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(raw);
  uint32_t* tmemAt = reinterpret_cast<uint32_t*>(raw + 256);
  volatile int* dead = reinterpret_cast<int*>(raw + 264);
  float* deltas = reinterpret_cast<float*>(raw + 512);
  const uint32_t tile0 = (smemAddr(raw) + 1024 + 1023) / 1024 * 1024, qTile = tile0, doTile = tile0 + F::kQBytes, kRing = tile0 + 2 * F::kQBytes,
                 vRing = kRing + F::kKSlots * F::kTileBytes;
  const auto bar = [&](int i) { return smemAddr(bars) + 8 * i; };
  const int warp = uniform(int(threadIdx.x) / 32), lane = threadIdx.x % 32;
  const int q0 = (int(gridDim.z) - 1 - int(blockIdx.z)) * kTile, h = blockIdx.x / split, rank = blockIdx.x % split, b = blockIdx.y, kv = h / (a.heads / a.kvHeads);
  // tiles of keys that the queries see, and this block's part of them
  const int keys = keysOf(a, b), all = colTiles<P>(seenBy(a, min(q0 + kTile, a.sq) - 1, keys));
  const int begun = int((long long)all * rank / split);

  const auto loadKeys = [&](int j) {
    const int ks = j % F::kKSlots;
    barExpect(bar(F::kKFull + ks), F::kTileBytes);
    loadTile<P, kCols>(kRing + ks * F::kTileBytes, &a.k, bar(F::kKFull + ks), (begun + j) * kCols, kv, b);
  };
  const auto loadValues = [&](int j) {
    const int vs = j % F::kVSlots;
    barExpect(bar(F::kVFull + vs), F::kTileBytes);
    loadTile<P, kCols>(vRing + vs * F::kTileBytes, &a.v, bar(F::kVFull + vs), (begun + j) * kCols, kv, b);
  };
  if (warp == kLoadWarp) {
    if (lane == 0) {
      for (int i = 0; i < F::kBars; i++) barInit(bar(i), i == F::kDsFull ? kComputeWarps : 1);
      dead[0] = isVoid(a.status), dead[1] = 0;
      fenceBarInit();
      fenceAsyncShared();
    }
    __syncwarp();
  }
  const uint32_t tmem = begin<P>(warp, tmemAt), dp = tmem + 2 * kCols, dq = tmem + 3 * kCols;
  if (warp == kMmaWarp) dead[1] = 1;
  const int n = uniform(*dead) ? 0 : int((long long)all * (rank + 1) / split) - begun;
  if constexpr (kLifted<T>) waitForPrevious();  // for the bounds
  // The next kernel's blocks may come now, before this one's allocation even: shared memory keeps any that
  // would need this block's tensor memory off the SM until it has left.
  letNextStart();

  if (warp == kLoadWarp) {
    L::other();
    if (lane == 0 && n) {
      barExpect(bar(F::kQFull), 2 * F::kQBytes);
      loadTile<P, kTile>(qTile, &a.q, bar(F::kQFull), q0, h, b);
      loadKeys(0);
      loadTile<P, kTile>(doTile, &a.dout, bar(F::kQFull), q0, h, b);
      loadValues(0);
      for (int j = 1; j < n; j++) {
        if (j >= F::kKSlots) barWait(bar(F::kKEmpty + j % F::kKSlots), (j / F::kKSlots - 1) & 1, dead);
        loadKeys(j);
        if (j >= F::kVSlots) barWait(bar(F::kVEmpty + j % F::kVSlots), (j / F::kVSlots - 1) & 1, dead);
        loadValues(j);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    L::other();
    const bool leader = electOne();
    const int steps = (a.d + 15) / 16;
    const uint32_t scores = mmaShape<T>(kCols, false), back = mmaShape<T>(steps * 16, true);
    const auto score = [&](int j) {  // S of key tile j
      const int ks = j % F::kKSlots;
      const uint32_t kTileAt = kRing + ks * F::kTileBytes;
      barWait(bar(F::kKFull + ks), j / F::kKSlots & 1, dead);
      if ((begun + j + 1) * kCols > keys && keys < a.sk) clearRows<P>(kTileAt, keys - (begun + j) * kCols);
      if (leader) {
        mmaTiles<P>(tmem + (j & 1) * kCols, qTile, kTileAt, scores, steps);
        mmaCommit(bar(F::kSFull + (j & 1)));
      }
    };
    const auto gradient = [&](int j) {  // dP of key tile j
      const int vs = j % F::kVSlots;
      barWait(bar(F::kVFull + vs), j / F::kVSlots & 1, dead);
      if (leader) {
        mmaTiles<P>(dp, doTile, vRing + vs * F::kTileBytes, scores, steps);
        mmaCommit(bar(F::kDpFull));
        if (j + F::kVSlots < n) mmaCommit(bar(F::kVEmpty + vs));
      }
    };
    if (n) {
      barWait(bar(F::kQFull), 0, dead);
      score(0);
      gradient(0);
      if (n > 1) score(1);
      for (int j = 0; j < n; j++) {
        barWait(bar(F::kDsFull), j & 1, dead);
        tcAfter();
        if (j + 1 < n) gradient(j + 1);
        if (leader) {
          const int ks = j % F::kKSlots;
          mmaTmemTile<kCols, kHalf>(dq, tmem + (j & 1) * kCols, kRing + ks * F::kTileBytes, back, j > 0);
          if (j + F::kKSlots < n) mmaCommit(bar(F::kKEmpty + ks));
          if (j == n - 1) mmaCommit(bar(F::kDone));
        }
        if (j + 2 < n) score(j + 2);
        __syncwarp();
      }
    }
  } else if (warp < kComputeWarps) {
    L::compute();
    const int half = warp / 4, row = warp % 4 * 32 + lane, i = q0 + row;
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const bool live = i < a.sq;
    const long long stat = ((long long)b * a.heads + h) * a.sq + i;
    const float c = a.scale * kLog2e;
    const long long at = (((long long)b * a.sq + i) * a.heads + h) * a.d;
    if (half == 0) {
      float sum = 0.f;
      if (live && all > 1) {
        const T *o = static_cast<const T*>(a.out) + at, *g = static_cast<const T*>(a.doutPtr) + b * a.doutB + i * a.doutS + h * a.doutH;
        for (int k = 0; k < a.d; k += 8) {
          float2 x[4], y[4], part = {0.f, 0.f};
          pairs(*reinterpret_cast<const Vec8<T>*>(o + k), x);
          pairs(*reinterpret_cast<const Vec8<T>*>(g + k), y);
#pragma unroll
          for (int u = 0; u < 4; u++) part = fma2(x[u], y[u], part);
          sum += part.x + part.y;
        }
      }
      if (live && all != 1 && rank == 0) a.delta[stat] = sum;
      deltas[row] = sum;
    }
    const float lift = liftOf<T>(a, b, kv);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    float delta = deltas[row];
    // a row that sees nothing, or lies behind the last query, has no probabilities
    float l = live ? a.lse[stat] * -kLog2e : -INFINITY;
    if (l == INFINITY) l = -INFINITY;
    const int seen = live ? seenBy(a, i, keys) : 0, whole = seenBy(a, q0, keys) / kCols;
    for (int j = 0; j < n; j++) {
      const uint32_t s = tmem + (j & 1) * kCols + half * kHalf + lanes;
      barWait(bar(F::kSFull + (j & 1)), j / 2 & 1, dead);
      tcAfter();
      uint32_t x[kHalf];
      tmemLoad<kHalf>(s, x);
      tmemWaitLoad();
#pragma unroll
      for (int k = 0; k < kHalf; k += 2) {
        const float2 e = fma2({__uint_as_float(x[k]), __uint_as_float(x[k + 1])}, {c, c}, {l, l});
        x[k] = __float_as_uint(exp2Fast(e.x)), x[k + 1] = __float_as_uint(exp2Fast(e.y));
      }
      barWait(bar(F::kDpFull), j & 1, dead);
      tcAfter();
      uint32_t y[kHalf], ds[kHalf / 2];
      tmemLoad<kHalf>(dp + half * kHalf + lanes, y);
      tmemWaitLoad();
      const int left = seen - (begun + j) * kCols - half * kHalf;
      if (all == 1) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kHalf; k++)
          if (k < left) sum += __uint_as_float(x[k]) * __uint_as_float(y[k]);
        // both halves' parts, always in the same order
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (half) deltas[row] = sum;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (!half) {
          sum += deltas[row];
          if (live) a.delta[stat] = sum;
          deltas[row] = sum;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        delta = deltas[row];
      }
      const float minus = kLifted<T> ? -delta * lift : -delta;
      const auto gradients = [&](auto masked) {
#pragma unroll
        for (int k = 0; k < kHalf; k += 2) {
          float2 g = lifted<T>({__uint_as_float(y[k]), __uint_as_float(y[k + 1])}, lift, {minus, minus});
          g = mul2({__uint_as_float(x[k]), __uint_as_float(x[k + 1])}, g);
          if (decltype(masked)::value) {
            g.x = k < left ? g.x : 0.f;
            g.y = k + 1 < left ? g.y : 0.f;
          }
          ds[k / 2] = pack2<T>(g.x, g.y);
        }
      };
      if (begun + j < whole) gradients(std::false_type());
      else gradients(std::true_type());
      tmemStore<kHalf / 2>(s, ds);
      tmemWaitStore();
      tcBefore();
      __syncwarp();
      if (lane == 0) barArrive(bar(F::kDsFull));
    }
    if (n) {
      barWait(bar(F::kDone), 0, dead);
      tcAfter();
    }
    if (*dead && half == 0 && seen > 0) a.delta[stat] = NAN;
    if constexpr (kSplit)
      leaveRow<L::kHeadCols, L::kHeadCols / 2>(kRing, row, dq + lanes, half * L::kHeadCols / 2, n > 0, dead);
    else
      storeRows<T, L::kHeadCols / 2>(static_cast<T*>(a.dq) + (((long long)b * a.sq + i - lane) * a.heads + h) * a.d, (int64_t)a.heads * a.d, a.sq - (i - lane),
                                     dq + lanes, half * L::kHeadCols / 2, a.d, factor(seen > 0, a.scale * reciprocal(lift), dead), n > 0, qTile + warp * (F::kQBytes / 8));
  } else {
    L::other();
  }
  if constexpr (kSplit) {
    clusterSync();
    if (warp < kComputeWarps) {
      const int rows = kTile / split, chunks = a.d / 8, count = rows * chunks;
      const float by = a.scale * reciprocal(liftOf<T>(a, b, kv));
      for (int k = threadIdx.x; k < count; k += kComputeWarps * 32) {
        const int row = rank * rows + k / chunks, chunk = k % chunks, i = q0 + row;
        float sum[8] = {};
        for (int r = 0; r < split; r++) addRow8<L::kHeadCols>(kRing, row, chunk, r, 1.f, sum);
        if (i < a.sq)
          *reinterpret_cast<uint4*>(static_cast<T*>(a.dq) + (((long long)b * a.sq + i) * a.heads + h) * a.d + chunk * 8) =
              rounded8<T>(reinterpret_cast<const uint32_t*>(sum), seenBy(a, i, keys) > 0 ? by : 0.f);
      }
    }
    clusterSync();  // nobody leaves while its sums are read
  }
  finish<P>(a, tmem, dead);
}

// ------------------------------------------------------------------ backward, keys
// A block owns 128 keys of one key head and goes through the query tiles of all query heads of
// its group:  S^T = K Q^T, dP^T = V dout^T, then dv += P^T dout and dk += dS^T Q.  While the warps
// make P, the matrix units do the last tile's dk and this one's dP; while they make dS, dv and
// the next scores.
template <class T, int P> struct Keys {
  static constexpr int kStages = P == 2 ? 2 : 4;
  static constexpr uint32_t kTileBytes = Tiling<P>::kColTile, kKBytes = Tiling<P>::kRowTile;
  static_assert(2 * kStages * kTileBytes >= 2 * kTile * Tiling<P>::kHeadCols * 4, "the sums of a shared tile fit the ring");
  static constexpr size_t kShared = kSharedBytes + 1024 + 2 * kKBytes + 2 * kStages * kTileBytes;
  enum { kKvFull = 0, kFull = 1, kEmpty = kFull + kStages, kSFull = kEmpty + kStages, kDpFull, kPFull, kDsFull, kDone, kBars };
};

template <class T, int P, bool kSplit> __global__ void __launch_bounds__(Tiling<P>::kThreads, Tiling<P>::kBlocks) keyKernel(const __grid_constant__ Args a) {
  using F = Keys<T, P>;
  using L = Tiling<P>;
  constexpr int kCols = L::kCols, kHalf = L::kHalf;
  static_assert(F::kBars <= 32 && F::kStages <= 4, "barriers");
  extern __shared__ char raw[];
  const int split = kSplit ? a.split : 1;
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const uint32_t kTileAt = (smemAddr(raw) + kSharedBytes + 1023) / 1024 * 1024, vTileAt = kTileAt + F::kKBytes, ring = vTileAt + F::kKBytes;
  const auto bar = [&](int i) { return smemAddr(sh.bars) + 8 * i; };
  volatile int* dead = sh.dead;
  const int warp = uniform(int(threadIdx.x) / 32), lane = threadIdx.x % 32;
  const int j0 = blockIdx.z * kTile, kv = blockIdx.x / split, rank = blockIdx.x % split, b = blockIdx.y, group = a.heads / a.kvHeads;
  const int keys = keysOf(a, b);
  const int first = a.causal ? max(0, j0 - (a.sk - a.sq)) / kCols : 0;  // first query tile that sees a key of this one
  const int each = j0 < keys ? max(0, colTiles<P>(a.sq) - first) : 0, all = each * group;
  // this block's part of the tiles
  const int begun = int((long long)all * rank / split);

  if (warp == kLoadWarp) {
    if (lane == 0) {
      for (int i = 0; i < F::kBars; i++)
        barInit(bar(i), i == F::kPFull || i == F::kDsFull ? kComputeWarps : i >= F::kFull && i < F::kEmpty ? 33 : 1);
      dead[0] = isVoid(a.status), dead[1] = 0;
      fenceBarInit();
      fenceAsyncShared();
    }
    __syncwarp();
  }
  const uint32_t tmem = begin<P>(warp, &sh.tmem), s = tmem, dp = tmem + kCols, dv = tmem + 2 * kCols, dk = dv + L::kHeadCols;
  if (warp == kMmaWarp) dead[1] = 1;
  const int n = uniform(*dead) ? 0 : int((long long)all * (rank + 1) / split) - begun;
  waitForPrevious();  // for delta

  if (warp == kLoadWarp) {
    L::other();
    if (lane == 0 && n) {
      barExpect(bar(F::kKvFull), 2 * F::kKBytes);
      loadTile<P, kTile>(kTileAt, &a.k, bar(F::kKvFull), j0, kv, b);
      loadTile<P, kTile>(vTileAt, &a.v, bar(F::kKvFull), j0, kv, b);
    }
    const float lift = kLifted<T> ? liftOf<T>(a, b, kv) * kProbabilityDrop : 1.f;
    for (int it = 0, h = kv * group + (n ? begun / each : 0), qt = n ? begun % each : 0; it < n; it++) {
      const int st = it % F::kStages, turn = it / F::kStages, q0 = (first + qt) * kCols;
      const long long stat = ((long long)b * a.heads + h) * a.sq;
      float l[kCols / 32], d[kCols / 32];
#pragma unroll
      for (int u = 0; u < kCols / 32; u++) {
        const int i = q0 + u * 32 + lane;
        l[u] = i < a.sq ? a.lse[stat + i] * -kLog2e : -INFINITY;
        if (l[u] == INFINITY) l[u] = -INFINITY;
        d[u] = i < a.sq ? -a.delta[stat + i] : 0.f;
        if constexpr (kLifted<T>) l[u] += kProbabilityLift, d[u] *= lift;
      }
      if (turn) barWait(bar(F::kEmpty + st), (turn - 1) & 1, dead);
      if (lane == 0) {
        const uint32_t q = ring + 2 * st * F::kTileBytes;
        barExpect(bar(F::kFull + st), 2 * F::kTileBytes);
        loadTile<P, kCols>(q, &a.q, bar(F::kFull + st), q0, h, b);
        loadTile<P, kCols>(q + F::kTileBytes, &a.dout, bar(F::kFull + st), q0, h, b);
      }
#pragma unroll
      for (int u = 0; u < kCols / 32; u++) sh.stats[st][0][u * 32 + lane] = l[u], sh.stats[st][1][u * 32 + lane] = d[u];
      barArrive(bar(F::kFull + st));
      if (++qt == each) qt = 0, h++;
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    L::other();
    const bool leader = electOne();
    const int steps = (a.d + 15) / 16;
    const uint32_t scores = mmaShape<T>(kCols, false), back = mmaShape<T>(steps * 16, true);
    if (n) {
      barWait(bar(F::kKvFull), 0, dead);
      for (int it = -1; it < n; it++) {
        const int st = (it + F::kStages) % F::kStages, next = (it + 1) % F::kStages;
        const uint32_t q = ring + 2 * st * F::kTileBytes, qn = ring + 2 * next * F::kTileBytes;
        if (it >= 0) {
          barWait(bar(F::kPFull), it & 1, dead);
          tcAfter();
          if (leader) mmaTmemTile<kCols, kHalf>(dv, s, q + F::kTileBytes, back, it > 0);
        }
        if (it + 1 < n) {
          barWait(bar(F::kFull + next), (it + 1) / F::kStages & 1, dead);
          if (leader) {
            mmaTiles<P>(s, kTileAt, qn, scores, steps);
            mmaCommit(bar(F::kSFull));
          }
        }
        if (it >= 0) {
          barWait(bar(F::kDsFull), it & 1, dead);
          tcAfter();
          if (leader) {
            mmaTmemTile<kCols, kHalf>(dk, dp, q, back, it > 0);
            if (it + F::kStages < n) mmaCommit(bar(F::kEmpty + st));
            if (it == n - 1) mmaCommit(bar(F::kDone));
          }
        }
        if (it + 1 < n && leader) {
          mmaTiles<P>(dp, vTileAt, qn + F::kTileBytes, scores, steps);
          mmaCommit(bar(F::kDpFull));
        }
        __syncwarp();
      }
    }
  } else if (warp < kComputeWarps) {
    L::compute();
    const int half = warp / 4;
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const float c = a.scale * kLog2e;
    // Scores are read in blocks of 16 lanes by 8 columns: a thread has two columns of each block,
    // whose statistics it reads from shared memory once for four rows.  (With a row to a thread
    // every statistic went to every thread, and reading them took as long as the exponentials.)
    constexpr int kBlocks8 = kHalf / 8, kRegs = kHalf / 2;
    const float whole = liftOf<T>(a, b, kv), lift = kLifted<T> ? whole * kProbabilityDrop : 1.f;
    const int row0 = warp % 4 * 32 + lane / 4, col0 = lane % 4 * 2;
    for (int it = 0, qt = n ? begun % each : 0; it < n; it++) {
      const int st = it % F::kStages, q0 = (first + qt) * kCols;
      if (++qt == each) qt = 0;
      const float* l = sh.stats[st][0] + half * kHalf + col0;
      const float* d = sh.stats[st][1] + half * kHalf + col0;
      // first column of the half that sees key j0 + row, less the thread's first
      const int edge = a.causal ? j0 - (a.sk - a.sq) - q0 - half * kHalf - col0 : -kTile - kCols;
      const bool some = j0 + kTile > keys || (a.causal && j0 + kTile - 1 > q0 + a.sk - a.sq);
      const auto from = [&](int row) { return j0 + row < keys ? edge + row : kCols; };
      barWait(bar(F::kFull + st), it / F::kStages & 1, dead);
      barWait(bar(F::kSFull), it & 1, dead);
      tcAfter();
      uint32_t x[2][kRegs];
      tmemLoadBlocks<kRegs>(s + half * kHalf + lanes, x[0]);
      tmemLoadBlocks<kRegs>(s + half * kHalf + lanes + (16 << 16), x[1]);
      tmemWaitLoad();
      const auto probabilities = [&](auto masked) {
#pragma unroll
        for (int k = 0; k < kBlocks8; k++) {
          const float2 ls = *reinterpret_cast<const float2*>(l + k * 8);
#pragma unroll
          for (int u = 0; u < 4; u++) {  // rows row0 + 8 u
            uint32_t* v = x[u / 2] + k * 4 + u % 2 * 2;
            float2 e = fma2({__uint_as_float(v[0]), __uint_as_float(v[1])}, {c, c}, ls);
            e.x = exp2Fast(e.x), e.y = exp2Fast(e.y);
            if (decltype(masked)::value) {
              e.x = k * 8 >= from(row0 + u * 8) ? e.x : 0.f;
              e.y = k * 8 + 1 >= from(row0 + u * 8) ? e.y : 0.f;
            }
            v[0] = __float_as_uint(e.x), v[1] = __float_as_uint(e.y);
          }
        }
      };
      if (some) probabilities(std::true_type());
      else probabilities(std::false_type());
      const auto store = [&](uint32_t at) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          uint32_t o[kRegs / 2];
#pragma unroll
          for (int k = 0; k < kRegs / 2; k++) o[k] = pack2<T>(__uint_as_float(x[r][2 * k]), __uint_as_float(x[r][2 * k + 1]));
          tmemStoreBlocks<kRegs / 2>(at + half * kHalf + lanes + (r * 16 << 16), o);
        }
        tmemWaitStore();
        tcBefore();
        __syncwarp();
      };
      store(s);
      if (lane == 0) barArrive(bar(F::kPFull));

      barWait(bar(F::kDpFull), it & 1, dead);
      tcAfter();
      uint32_t y[2][kRegs];
      tmemLoadBlocks<kRegs>(dp + half * kHalf + lanes, y[0]);
      tmemLoadBlocks<kRegs>(dp + half * kHalf + lanes + (16 << 16), y[1]);
      tmemWaitLoad();
      const auto gradients = [&](auto masked) {
#pragma unroll
        for (int k = 0; k < kBlocks8; k++) {
          const float2 ds = *reinterpret_cast<const float2*>(d + k * 8);
#pragma unroll
          for (int u = 0; u < 4; u++) {
            uint32_t *v = x[u / 2] + k * 4 + u % 2 * 2, *w = y[u / 2] + k * 4 + u % 2 * 2;
            float2 g = lifted<T>({__uint_as_float(w[0]), __uint_as_float(w[1])}, lift, ds);
            g = mul2({__uint_as_float(v[0]), __uint_as_float(v[1])}, g);
            if (decltype(masked)::value) {
              g.x = k * 8 >= from(row0 + u * 8) ? g.x : 0.f;
              g.y = k * 8 + 1 >= from(row0 + u * 8) ? g.y : 0.f;
            }
            v[0] = __float_as_uint(g.x), v[1] = __float_as_uint(g.y);
          }
        }
      };
      if (some) gradients(std::true_type());
      else gradients(std::false_type());
      store(dp);
      if (lane == 0) barArrive(bar(F::kDsFull));
    }
    const int row = warp % 4 * 32 + lane, j = j0 + row;
    const bool counts = j < keys;
    if (n) {
      barWait(bar(F::kDone), 0, dead);
      tcAfter();
    }
    if constexpr (!kSplit) {
      const int jw = j - lane;  // the warp's first row
      const long long at = (((long long)b * a.sk + jw) * a.kvHeads + kv) * a.d;
      const int64_t stride = (int64_t)a.kvHeads * a.d;
      storeRows<T, L::kHeadCols / 2>(static_cast<T*>(a.dv) + at, stride, a.sk - jw, dv + lanes, half * L::kHeadCols / 2, a.d, factor(counts, kLifted<T> ? kProbabilityDrop : 1.f, dead), n > 0,
                                     vTileAt + warp * (F::kKBytes / 8));
      storeRows<T, L::kHeadCols / 2>(static_cast<T*>(a.dk) + at, stride, a.sk - jw, dk + lanes, half * L::kHeadCols / 2, a.d, factor(counts, a.scale * reciprocal(whole), dead), n > 0,
                                     kTileAt + warp * (F::kKBytes / 8));
    } else {
      // the tiles of the ring are done with: dv, then dk, in 32 bits
      leaveRow<L::kHeadCols, L::kHeadCols / 2>(ring, row, dv + lanes, half * L::kHeadCols / 2, n > 0, dead);
      leaveRow<L::kHeadCols, L::kHeadCols / 2>(ring + kTile * L::kHeadCols * 4, row, dk + lanes, half * L::kHeadCols / 2, n > 0, dead);
    }
  } else {
    L::other();
  }
  if constexpr (kSplit) {
    clusterSync();
    if (warp < kComputeWarps) {
      const float byV = kLifted<T> ? kProbabilityDrop : 1.f, byK = a.scale * reciprocal(liftOf<T>(a, b, kv));
      const int rows = kTile / split, row0 = rank * rows, chunks = a.d / 8, count = 2 * rows * chunks;
      for (int i = threadIdx.x; i < count; i += kComputeWarps * 32) {
        const int which = i / (rows * chunks), row = row0 + i / chunks % rows, c = i % chunks, j = j0 + row;
        float sum[8] = {};
        for (int r = 0; r < split; r++) addRow8<L::kHeadCols>(ring + which * kTile * L::kHeadCols * 4, row, c, r, 1.f, sum);
        if (j >= a.sk) continue;
        T* out = static_cast<T*>(which ? a.dk : a.dv) + (((long long)b * a.sk + j) * a.kvHeads + kv) * a.d + c * 8;
        *reinterpret_cast<uint4*>(out) = rounded8<T>(reinterpret_cast<const uint32_t*>(sum), j >= keys ? 0.f : which ? byK : byV);
      }
    }
    clusterSync();  // nobody leaves while its sums are read
  }
  finish<P>(a, tmem, dead);
}

// ------------------------------------------------------------------ host
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
  static const Encode f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return f;
}

int makeMap(CUtensorMap* map, const char* name, const tcpxbHeads& x, int b, int s, int heads, int d, int rows, int dtype) {
  std::memset(map, 0, sizeof(*map));
  if ((long long)b * s == 0) return TCPXB_T_OK;  // nothing is loaded
  const Encode encode = encoder();
  if (!encode) return fail(TCPXB_T_CUDA, "the driver has no tensor maps");
  const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(s), cuuint64_t(heads), cuuint64_t(b)};
  cuuint64_t strides[3] = {cuuint64_t(x.stride_s) * 2, cuuint64_t(x.stride_h) * 2, cuuint64_t(x.stride_b) * 2};
  for (int i = 0; i < 3; i++)
    if (dims[i + 1] == 1) strides[i] = 256;  // of no influence
  const cuuint32_t box[4] = {64, cuuint32_t(rows), 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, dtype == TCPXB_T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, x.ptr, dims, strides, box,
                            ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TCPXB_T_OK : fail(TCPXB_T_INVALID, "%s cannot be loaded in tiles (driver error %d): its strides are out of range", name, int(r));
}

bool stridesOk(const tcpxbHeads& x, int b, int s, int heads) {
  return headsOk(x, 2) && (b == 1 || x.stride_b > 0) && (s == 1 || x.stride_s > 0) && (heads == 1 || x.stride_h > 0);
}

int check(const tcpxbAttention* a, bool backward) {
  if (!a) return fail(TCPXB_T_INVALID, "null argument");
  if (a->b < 0 || a->sq < 0 || a->sk < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->d < 8 || a->d > kMaxD || a->d % 8)
    return fail(TCPXB_T_INVALID, "bad shape: b %d sq %d sk %d heads %d/%d d %d", a->b, a->sq, a->sk, a->heads, a->kv_heads, a->d);
  if (a->b > 65535 || a->heads > 65535 || a->sq > 65535 * kTile || a->sk > 65535 * kTile)
    return fail(TCPXB_T_INVALID, "at most 65535 batches, heads and tiles of 128 tokens: b %d heads %d sq %d sk %d", a->b, a->heads, a->sq, a->sk);
  if (a->dtype != TCPXB_T_BF16 && a->dtype != TCPXB_T_F16) return fail(TCPXB_T_INVALID, "attention takes bf16 and fp16, not type %d", a->dtype);
  if (!(a->scale > 0.f) || a->scale > 1e30f) return fail(TCPXB_T_INVALID, "scale has to be finite and above zero");
  const bool queries = (long long)a->b * a->sq > 0, keys = (long long)a->b * a->sk > 0;
  if (queries && (!stridesOk(a->q, a->b, a->sq, a->heads) || !a->out || !a->lse))
    return fail(TCPXB_T_INVALID, "q, out or lse is null, off the 16-byte boundary or broadcast");
  if (keys && (!stridesOk(a->k, a->b, a->sk, a->kv_heads) || !stridesOk(a->v, a->b, a->sk, a->kv_heads)))
    return fail(TCPXB_T_INVALID, "k or v is null, off the 16-byte boundary or broadcast");
  if (backward && queries && a->dtype == TCPXB_T_F16 && (!a->bounds || reinterpret_cast<uintptr_t>(a->bounds) % 8))
    return fail(TCPXB_T_INVALID, "fp16 gradients need `bounds`, on an 8-byte boundary");
  if (backward && ((queries && (!stridesOk(a->dout, a->b, a->sq, a->heads) || !a->dq || !a->delta)) || (keys && (!a->dk || !a->dv))))
    return fail(TCPXB_T_INVALID, "dout, dq, dk, dv or delta is null, off the 16-byte boundary or broadcast");
  return TCPXB_T_OK;
}

int makeArgs(const tcpxbAttention& a, bool backward, int rows, Args* x) {
  int rc = makeMap(&x->q, "q", a.q, a.b, a.sq, a.heads, a.d, rows, a.dtype);
  if (!rc) rc = makeMap(&x->k, "k", a.k, a.b, a.sk, a.kv_heads, a.d, rows, a.dtype);
  if (!rc) rc = makeMap(&x->v, "v", a.v, a.b, a.sk, a.kv_heads, a.d, rows, a.dtype);
  if (!rc && backward) rc = makeMap(&x->dout, "dout", a.dout, a.b, a.sq, a.heads, a.d, rows, a.dtype);
  if (rc) return rc;
  x->out = x->o = a.out;
  x->doutPtr = a.dout.ptr;
  x->doutB = a.dout.stride_b, x->doutS = a.dout.stride_s, x->doutH = a.dout.stride_h;
  x->vPtr = a.v.ptr, x->vB = a.v.stride_b, x->vS = a.v.stride_s, x->vH = a.v.stride_h;
  x->bounds = nullptr, x->parts = 0;
  x->dq = a.dq, x->dk = a.dk, x->dv = a.dv, x->lse = a.lse, x->delta = a.delta;
  x->keyLengths = a.key_lengths, x->status = a.status;
  x->b = a.b, x->sq = a.sq, x->sk = a.sk, x->heads = a.heads, x->kvHeads = a.kv_heads, x->d = a.d, x->causal = a.causal, x->scale = a.scale;
  return TCPXB_T_OK;
}

// Once for each kernel and device the block's shared memory is allowed; more than 64 devices would only ask again.
template <void (*kKernel)(Args)> int allow(size_t shared, int device, const char* what) {
  static std::atomic<uint64_t> allowed{0};
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return TCPXB_T_OK;
  const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
  if (e != cudaSuccess) return fail(TCPXB_T_CUDA, "%s: %s", what, cudaGetErrorString(e));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return TCPXB_T_OK;
}

// The kernel, or its form for clusters where `a.split` blocks share a tile; `behind` another kernel of this call.
template <void (*kKernel)(Args), void (*kClusters)(Args)>
int launch(bool behind, dim3 grid, int threads, size_t shared, const Args& a, int device, cudaStream_t s, const char* what) {
  if (const int rc = a.split == 1 ? allow<kKernel>(shared, device, what) : allow<kClusters>(shared, device, what)) return rc;
  cudaLaunchAttribute attributes[2];
  cudaLaunchConfig_t config = {};
  config.gridDim = grid, config.blockDim = dim3(threads), config.dynamicSmemBytes = shared, config.stream = s;
  config.attrs = attributes, config.numAttrs = 0;
  if (a.split > 1) {
    cudaLaunchAttribute& x = attributes[config.numAttrs++];
    x.id = cudaLaunchAttributeClusterDimension;
    x.val.clusterDim.x = unsigned(a.split), x.val.clusterDim.y = x.val.clusterDim.z = 1;
  }
  if (behind) {
    cudaLaunchAttribute& x = attributes[config.numAttrs++];
    x.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    x.val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchKernelEx(&config, a.split == 1 ? kKernel : kClusters, a);
  return launched(what);
}

template <class T, int P> int run(const tcpxbAttention& a, bool backward, cudaStream_t s) {
  if (const int rc = use(a.device)) return rc;
  const int device = a.device;
  Args x;
  if (const int rc = makeArgs(a, backward, Tiling<P>::kCols, &x)) return rc;
  constexpr int kCols = Tiling<P>::kCols;
  // A cluster where all blocks find room at the same time, with at least four (gradients of keys) or eight
  // tiles for each.  2 x 512 tokens, 16/4 heads of 64, causal, gradients of keys: 32 tiles in one block 31.6 us, 8 in each of four
  // 16.2 us; 1000 tokens, 8/1 heads of 128: 99.7 us, in fours 37.1 us, in eights 28.7 us.  Where blocks come
  // in several rounds a cluster's overhead, about six tiles of 64, is lost (512 blocks 163 us, in fours
  // 211 us), and eights do not pack: 256 of their blocks take 24.5 us for the first example.
  const auto splitFor = [](long long blocks, long long tiles, int least) {
    int split = 1;
    while (split < 8 && blocks * split * 2 <= (split == 4 ? 148 : 148 * Tiling<P>::kBlocks) && tiles / (split * 2) >= least) split *= 2;
    return split;
  };
  const long long tilesOfKeys = (a.sk + kTile - 1) / kTile, colsOfKeys = (a.sk + kCols - 1) / kCols;
  const long long tilesOfQueries = (a.sq + kTile - 1) / kTile, pairsOfQueries = (tilesOfQueries + 1) / 2;
  if (!backward) {
    if (!a.b || !a.sq) return TCPXB_T_OK;
    x.split = splitFor(pairsOfQueries * a.heads * a.b, colsOfKeys, 8);
    return launch<forwardKernel<T, P, false>, forwardKernel<T, P, true>>(false, dim3(a.heads * x.split, a.b, unsigned(pairsOfQueries)), Tiling<P>::kThreads, Forward<T, P>::kShared, x, device, s,
                                       "attention forward");
  }
  if (a.b && a.sq) {
    if constexpr (kLifted<T>) {
      x.bounds = reinterpret_cast<const float2*>(a.bounds);
      const long long pairs = (long long)a.kv_heads * a.b;
      x.parts = int(std::clamp<long long>(2 * 148 / pairs, 1, kParts));
      boundsKernel<T, P><<<dim3(x.parts, a.kv_heads, a.b), kBoundsThreads, 0, s>>>(x, reinterpret_cast<float2*>(a.bounds));
      if (const int rc = launched("attention backward, bounds")) return rc;
    }
    x.split = splitFor(tilesOfQueries * a.heads * a.b, colsOfKeys, 8);
    if (const int rc = launch<queryKernel<T, P, false>, queryKernel<T, P, true>>(kLifted<T>, dim3(a.heads * x.split, a.b, unsigned(tilesOfQueries)), Tiling<P>::kThreads, Queries<T, P>::kShared, x,
                                                 device, s, "attention backward, queries"))
      return rc;
  }
  if (!a.b || !a.sk) return TCPXB_T_OK;
  x.split = splitFor(tilesOfKeys * a.kv_heads * a.b, (long long)(a.sq + kCols - 1) / kCols * (a.heads / a.kv_heads), 4);
  return launch<keyKernel<T, P, false>, keyKernel<T, P, true>>(a.b && a.sq, dim3(a.kv_heads * x.split, a.b, unsigned(tilesOfKeys)), Tiling<P>::kThreads, Keys<T, P>::kShared, x, device, s,
                                 "attention backward, keys");
}

int dispatch(const tcpxbAttention* a, bool backward, void* stream) {
  if (const int rc = check(a, backward)) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == TCPXB_T_BF16) return a->d <= 64 ? run<__nv_bfloat16, 1>(*a, backward, s) : run<__nv_bfloat16, 2>(*a, backward, s);
  return a->d <= 64 ? run<__half, 1>(*a, backward, s) : run<__half, 2>(*a, backward, s);
}

}  // namespace
}  // namespace tcpxb_train

using namespace tcpxb_train;

extern "C" int tcpxb_attention_forward(const tcpxbAttention* a, void* stream) { return dispatch(a, false, stream); }
extern "C" int tcpxb_attention_backward(const tcpxbAttention* a, void* stream) { return dispatch(a, true, stream); }
