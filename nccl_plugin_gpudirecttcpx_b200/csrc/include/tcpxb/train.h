// C ABI of the training step's device operators: attention forward and backward, per-head
// norms of queries and keys with the position rotation, and AdamW over many tensors.
//
// All functions return 0 on success or a negative tcpxbTrainError; the text of the last
// failure on the calling thread is available from tcpxb_train_last_error().  Work is queued
// on `stream`; nothing is allocated, copied to the host or kept between calls.
#ifndef TCPXB_TRAIN_H_
#define TCPXB_TRAIN_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum tcpxbTrainDtype {
  TCPXB_T_BF16 = 1,  // the codes of tcpxbDtype, where both have the type
  TCPXB_T_F32 = 2,
  TCPXB_T_F16 = 3,
} tcpxbTrainDtype;

typedef enum tcpxbTrainError {
  TCPXB_T_OK = 0,
  TCPXB_T_INVALID = -1,  // bad argument
  TCPXB_T_CUDA = -2,     // a CUDA call failed
} tcpxbTrainError;

const char* tcpxb_train_last_error(void);

// A [batch, tokens, heads, head size] tensor: head elements contiguous, the other strides in
// elements and multiples of 16 bytes (for attention above zero), base on a 16-byte boundary.
typedef struct tcpxbHeads {
  void* ptr;
  int64_t stride_b, stride_s, stride_h;
} tcpxbHeads;

// Attention of `sq` queries over `sk` keys.  Query i of batch b sees key j where
// j < key_lengths[b] (all keys without lengths; values outside [0, sk] count as the nearer end)
// and, with `causal`, j <= i + sk - sq.  `heads` is a multiple of `kv_heads`: query head h reads
// key head h / (heads / kv_heads).  A query that sees no key gets a zero row and lse = -infinity.
// What K and V hold behind a key length has no influence, NaN and infinities included.
typedef struct tcpxbAttention {
  tcpxbHeads q, k, v;     // bf16 or fp16
  void* out;              // [b, sq, heads, d], contiguous, type of q
  float* lse;             // [b, heads, sq]: natural logarithm of each row's sum of exponentials
  tcpxbHeads dout;        // backward only, as the rest
  void *dq, *dk, *dv;     // contiguous, type of q
  float* delta;           // [b, heads, sq] scratch
  const int32_t* key_lengths;  // [b] on the device, or null
  int32_t b, sq, sk, heads, kv_heads, d;  // d: a multiple of 8, at most 128
  float scale;            // above zero
  int32_t causal, dtype;
  int32_t device;         // that the tensors are on; becomes the calling thread's
  int32_t* status;        // a word on the device, or null: 3 (TCPXB_ST_TIMEOUT) where a bounded wait ran out.  The outputs are NaN then,
                          // and those of calls that find a 3 there: rows that see nothing apart
  float* bounds;          // [b, kv_heads, 64] scratch, on an 8-byte boundary; backward of fp16 only, not read else
} tcpxbAttention;

int tcpxb_attention_forward(const tcpxbAttention* a, void* stream);
int tcpxb_attention_backward(const tcpxbAttention* a, void* stream);

// n = x * rsqrt(mean(x^2) + eps) * w per head (n = x where w is null), then every pair
// (n[2i], n[2i+1]) is turned by the angle of its token's position.
typedef struct tcpxbNormRope {
  tcpxbHeads q, k;         // inputs
  const void *wq, *wk;     // [d] of type `dtype`, both or neither
  const float *cos, *sin;  // [positions, d / 2]
  const int64_t* pos;      // [b, s], or null for 0 .. s-1; a token outside the tables gets NaN rows
  void *q_out, *k_out;     // forward: contiguous
  tcpxbHeads dq_out, dk_out;  // backward: gradients of the outputs
  void *dq, *dk;           // contiguous
  void *dwq, *dwk;         // [d]
  float* partial;          // scratch: tcpxb_norm_rope_scratch_bytes()
  int32_t b, s, heads, kv_heads, d;  // d: a multiple of 8, at most 256
  int32_t positions;
  float eps;
  int32_t dtype, device;
} tcpxbNormRope;

size_t tcpxb_norm_rope_scratch_bytes(int d);
int tcpxb_norm_rope_forward(const tcpxbNormRope* a, void* stream);
int tcpxb_norm_rope_backward(const tcpxbNormRope* a, void* stream);

// One AdamW step.  States are 32-bit, or e4m3 with a 32-bit scale per 256 elements (the second
// one holds the root).  `step` counts the tensor's own updates and is advanced here.
#define TCPXB_ADAMW_BLOCK 256
typedef struct tcpxbAdamwTensor {
  void* p;
  const void* g;
  void *m, *v;
  float *m_scale, *v_scale;  // 8-bit states only
  float* master;             // 32-bit weights behind 16-bit ones, or null
  int32_t* step;
  int64_t n;
} tcpxbAdamwTensor;

typedef struct tcpxbAdamw {
  double lr, beta1, beta2, eps, weight_decay;
  float* grad_norm;        // device scalar: gradients are scaled by min(1, max_norm / (grad_norm + 1e-6)); null: not clipped
  float max_norm;
  int32_t compute_norm;    // write *grad_norm first, as tcpxb_grad_norm would
  int32_t state_bits, dtype, device;
  void* scratch;           // tcpxb_adamw_scratch_bytes()
} tcpxbAdamw;

size_t tcpxb_adamw_scratch_bytes(const tcpxbAdamwTensor* tensors, int count);
int tcpxb_adamw_step(const tcpxbAdamwTensor* tensors, int count, const tcpxbAdamw* a, void* stream);

// *norm = sqrt(sum of squares over all gradients (`g`, `n` of each tensor)).
size_t tcpxb_grad_norm_scratch_bytes(const tcpxbAdamwTensor* tensors, int count);
int tcpxb_grad_norm(const tcpxbAdamwTensor* tensors, int count, int dtype, int device, float* norm, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
#endif  // TCPXB_TRAIN_H_
