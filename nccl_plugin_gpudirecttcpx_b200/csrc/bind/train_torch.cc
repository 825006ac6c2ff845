// Tensors to the C ABI of the training step's operators: checks of arguments, outputs, scratch and
// streams, as a Python module.  It is compiled because a call's few microseconds of checks and
// allocations are what small calls consist of: through ctypes a toy model's AdamW step took 57 us
// and its attention, both ways, 39 us, of which the device needed 11 and 15; here 22 and 19.5 us.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <variant>
#include <vector>

#include "tcpxb/train.h"

namespace {

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using Maybe = std::optional<Tensor>;

void done(int rc, const char* what) { TORCH_CHECK(rc == TCPXB_T_OK, what, " failed (", rc, "): ", tcpxb_train_last_error()); }

int codeOf(ScalarType t) {
  return t == at::kBFloat16 ? TCPXB_T_BF16 : t == at::kFloat ? TCPXB_T_F32 : t == at::kHalf ? TCPXB_T_F16 : 0;
}

// All tensors are on one CUDA device, which becomes the current one for the call.
void onDevice(std::optional<c10::cuda::CUDAGuard>& guard, const Tensor& first, std::initializer_list<const Maybe*> rest) {
  bool ok = first.is_cuda();
  for (const Maybe* t : rest) ok = ok && (!t->has_value() || (*t)->device() == first.device());
  TORCH_CHECK_VALUE(ok, "all tensors have to be on one CUDA device");
  guard.emplace(first.device());
}
// A dual tensor of forward mode does not require gradients, so autograd's functions are passed by for it: its
// tangent would be lost without a word, which reads as a derivative of zero.
void noTangent(std::initializer_list<const Maybe*> tensors) {
  for (const Maybe* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->has_value() || !(*t)->_fw_grad(0).defined(), "forward-mode derivatives are not provided: gradients are taken backwards");
}
void* streamOf(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor make(const Tensor& like, at::IntArrayRef sizes, ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }
Tensor make(const Tensor& like, at::IntArrayRef sizes) { return make(like, sizes, like.scalar_type()); }

// The tensor itself where its head rows start on 16-byte boundaries and are not broadcast, else a
// contiguous copy that takes its place.
tcpxbHeads heads(Tensor& t) {
  const int64_t per = 16 / t.element_size();
  tcpxbHeads h;
  const auto describe = [&] {
    // the stride of a single entry is of no influence
    const auto stride = [&](int i) { return t.size(i) == 1 ? int64_t(16) : t.stride(i); };
    h = {t.data_ptr(), stride(0), stride(1), stride(2)};
    const bool rows = t.size(3) <= 1 || t.stride(3) == 1;
    return rows && reinterpret_cast<uintptr_t>(h.ptr) % 16 == 0 && h.stride_b > 0 && h.stride_s > 0 && h.stride_h > 0 && h.stride_b % per == 0 &&
           h.stride_s % per == 0 && h.stride_h % per == 0;
  };
  if (!describe()) {
    t = t.clone(at::MemoryFormat::Contiguous);
    describe();
  }
  return h;
}
Tensor aligned(const Tensor& t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ------------------------------------------------------------------ attention
struct Sizes {
  int64_t b, sq, sk, h, hk, d;
  double scale;
};

Sizes checkAttention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scale, const Maybe& lengths, const Maybe& status) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v have to be [batch, tokens, heads, head size], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  const auto type = q.scalar_type();
  TORCH_CHECK_TYPE((type == at::kBFloat16 || type == at::kHalf) && k.scalar_type() == type && v.scalar_type() == type,
                   "attention takes bfloat16 or float16 of one kind, got ", type, ", ", k.scalar_type(), ", ", v.scalar_type());
  Sizes s{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3), 0.0};
  TORCH_CHECK_VALUE(k.size(0) == s.b && k.size(3) == s.d && v.sizes() == k.sizes(), "shapes do not match: q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes());
  TORCH_CHECK_VALUE(s.h >= 1 && s.hk >= 1 && s.h % s.hk == 0, s.h, " query heads are no multiple of ", s.hk, " key heads");
  TORCH_CHECK_VALUE(s.d % 8 == 0 && s.d >= 8 && s.d <= 128, "the head size has to be a multiple of 8 up to 128, got ", s.d);
  TORCH_CHECK_VALUE(s.b <= 65535 && s.h <= 65535 && s.sq <= 65535 * 128 && s.sk <= 65535 * 128, "at most 65535 batches, heads and 128 x 65535 tokens: q ",
                    q.sizes(), ", k ", k.sizes());
  if (lengths) {
    TORCH_CHECK_TYPE(lengths->scalar_type() == at::kInt, "key_lengths has to be int32, got ", lengths->scalar_type());
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == s.b, "key_lengths has to be [", s.b, "], got ", lengths->sizes());
  }
  s.scale = scale.value_or(1.0 / std::sqrt(double(s.d)));
  TORCH_CHECK_VALUE(s.scale > 0 && s.scale < 1e30, "scale has to be finite and above zero, got ", s.scale);
  TORCH_CHECK_VALUE(!status || (status->scalar_type() == at::kInt && status->numel() >= 1 && status->is_contiguous()),
                    "status has to be a contiguous int32 tensor (ops.status_buffer())");
  return s;
}

tcpxbAttention describe(Tensor& q, Tensor& k, Tensor& v, const Sizes& s, bool causal, Maybe& lengths, const Maybe& status) {
  tcpxbAttention a = {};
  a.q = heads(q), a.k = heads(k), a.v = heads(v);
  if (lengths) lengths = lengths->contiguous(), a.key_lengths = lengths->data_ptr<int32_t>();
  if (status) a.status = status->data_ptr<int32_t>();
  a.b = int32_t(s.b), a.sq = int32_t(s.sq), a.sk = int32_t(s.sk), a.heads = int32_t(s.h), a.kv_heads = int32_t(s.hk), a.d = int32_t(s.d);
  a.scale = float(s.scale), a.causal = causal, a.dtype = codeOf(q.scalar_type()), a.device = q.get_device();
  return a;
}

std::tuple<Tensor, Tensor> attentionForward(Tensor q, Tensor k, Tensor v, bool causal, std::optional<double> scale, Maybe lengths, Maybe status) {
  const Sizes s = checkAttention(q, k, v, scale, lengths, status);
  std::optional<c10::cuda::CUDAGuard> guard;
  const Maybe mq = q, mk = k, mv = v;
  noTangent({&mq, &mk, &mv});
  onDevice(guard, q, {&mk, &mv, &lengths, &status});
  Tensor out = make(q, {s.b, s.sq, s.h, s.d}), lse = make(q, {s.b, s.h, s.sq}, at::kFloat);
  tcpxbAttention a = describe(q, k, v, s, causal, lengths, status);
  a.out = out.data_ptr(), a.lse = lse.data_ptr<float>();
  done(tcpxb_attention_forward(&a, streamOf(q)), "tcpxb_attention_forward");
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> attentionBackward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, bool causal,
                                                     std::optional<double> scale, Maybe lengths, Maybe status) {
  const Sizes s = checkAttention(q, k, v, scale, lengths, status);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"dout", dout}, {"out", out}}) {
    TORCH_CHECK_VALUE(t.sizes() == q.sizes(), name, " has to be ", q.sizes(), ", got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), name, " has to be ", q.scalar_type(), ", got ", t.scalar_type());
  }
  TORCH_CHECK_VALUE(lse.dim() == 3 && lse.size(0) == s.b && lse.size(1) == s.h && lse.size(2) == s.sq, "lse has to be [batch, heads, queries], got ", lse.sizes());
  TORCH_CHECK_TYPE(lse.scalar_type() == at::kFloat, "lse has to be float32, got ", lse.scalar_type());
  std::optional<c10::cuda::CUDAGuard> guard;
  const Maybe mq = q, mk = k, mv = v, mdout = dout, mout = out, mlse = lse;
  noTangent({&mq, &mk, &mv, &mdout, &mout, &mlse});
  onDevice(guard, q, {&mk, &mv, &mdout, &mout, &mlse, &lengths, &status});
  Tensor dq = make(q, {s.b, s.sq, s.h, s.d}), dk = make(q, {s.b, s.sk, s.hk, s.d}), dv = make(q, {s.b, s.sk, s.hk, s.d});
  Tensor delta = make(q, {s.b, s.h, s.sq}, at::kFloat), bounds;
  out = aligned(out), lse = lse.contiguous();
  tcpxbAttention a = describe(q, k, v, s, causal, lengths, status);
  a.dout = heads(dout);
  a.out = out.data_ptr(), a.lse = lse.data_ptr<float>(), a.delta = delta.data_ptr<float>();
  a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr();
  if (q.scalar_type() == at::kHalf) bounds = make(q, {s.b, s.hk, 64}, at::kFloat), a.bounds = bounds.data_ptr<float>();
  done(tcpxb_attention_backward(&a, streamOf(q)), "tcpxb_attention_backward");
  return {dq, dk, dv};
}

// ------------------------------------------------------------------ norms with rotation
// Sizes, type and eps; the weights' and positions' addresses come with the tensors that are kept for the call.
tcpxbNormRope checkNormRope(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Maybe& wq, const Maybe& wk, double eps,
                            const Maybe& positions) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "q and k have to be [batch, tokens, heads, head size], got ", q.sizes(), " and ", k.sizes());
  const auto type = q.scalar_type();
  TORCH_CHECK_TYPE(codeOf(type) && k.scalar_type() == type, "q and k have to be bfloat16, float16 or float32 of one kind, got ", type, " and ", k.scalar_type());
  const int64_t b = q.size(0), s = q.size(1), h = q.size(2), d = q.size(3), hk = k.size(2);
  TORCH_CHECK_VALUE(k.size(0) == b && k.size(1) == s && k.size(3) == d && h >= 1 && hk >= 1, "shapes do not match: q ", q.sizes(), ", k ", k.sizes());
  TORCH_CHECK_VALUE(d % 8 == 0 && d >= 8 && d <= 256, "the head size has to be a multiple of 8 up to 256, got ", d);
  TORCH_CHECK_VALUE(b < (1ll << 31) && s < (1ll << 31) && h + hk < (1ll << 31) && (b * s == 0 || b * s < (1ll << 31) / (h + hk)), "at most 2^31 - 1 rows: q ",
                    q.sizes(), ", k ", k.sizes());
  TORCH_CHECK_TYPE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin have to be float32, got ", cos.scalar_type(), " and ",
                   sin.scalar_type());
  TORCH_CHECK_VALUE(cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.size(1) == d / 2 && cos.size(0) < (1ll << 31), "cos and sin have to be [positions, ",
                    d / 2, "], got ", cos.sizes(), " and ", sin.sizes());
  if (positions) {
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kLong, "positions has to be int64, got ", positions->scalar_type());
    TORCH_CHECK_VALUE(positions->dim() == 2 && positions->size(0) == b && positions->size(1) == s, "positions has to be [", b, ", ", s, "], got ",
                      positions->sizes());
  } else {
    TORCH_CHECK_VALUE(cos.size(0) >= s, "the tables hold ", cos.size(0), " positions of ", s);
  }
  TORCH_CHECK_VALUE(wq.has_value() == wk.has_value(), "q_weight and k_weight come together");
  if (wq) {
    TORCH_CHECK_VALUE(wq->dim() == 1 && wk->dim() == 1 && wq->size(0) == d && wk->size(0) == d, "the weights have to be [", d, "], got ", wq->sizes(), " and ",
                      wk->sizes());
    TORCH_CHECK_TYPE(wq->scalar_type() == type && wk->scalar_type() == type, "the weights have to be ", type, ", got ", wq->scalar_type(), " and ",
                     wk->scalar_type());
  }
  TORCH_CHECK_VALUE(eps >= 0 && eps < INFINITY, "eps has to be finite and not below zero, got ", eps);
  tcpxbNormRope a = {};
  a.b = int32_t(b), a.s = int32_t(s), a.heads = int32_t(h), a.kv_heads = int32_t(hk), a.d = int32_t(d);
  a.positions = int32_t(cos.size(0)), a.eps = float(eps), a.dtype = codeOf(type);
  return a;
}

void describe(tcpxbNormRope& a, Tensor& cos, Tensor& sin, Maybe& wq, Maybe& wk, Maybe& positions) {
  cos = aligned(cos), sin = aligned(sin);
  a.cos = cos.data_ptr<float>(), a.sin = sin.data_ptr<float>(), a.device = cos.get_device();
  if (wq) wq = aligned(*wq), wk = aligned(*wk), a.wq = wq->data_ptr(), a.wk = wk->data_ptr();
  if (positions) positions = positions->contiguous(), a.pos = positions->data_ptr<int64_t>();
}

std::tuple<Tensor, Tensor> normRopeForward(Tensor q, Tensor k, Tensor cos, Tensor sin, Maybe wq, Maybe wk, double eps, Maybe positions) {
  tcpxbNormRope a = checkNormRope(q, k, cos, sin, wq, wk, eps, positions);
  std::optional<c10::cuda::CUDAGuard> guard;
  const Maybe mq = q, mk = k, mcos = cos, msin = sin;
  noTangent({&mq, &mk, &mcos, &msin, &wq, &wk});
  onDevice(guard, q, {&mk, &mcos, &msin, &wq, &wk, &positions});
  Tensor qOut = make(q, q.sizes()), kOut = make(k, k.sizes());
  describe(a, cos, sin, wq, wk, positions);
  a.q = heads(q), a.k = heads(k);
  a.q_out = qOut.data_ptr(), a.k_out = kOut.data_ptr();
  done(tcpxb_norm_rope_forward(&a, streamOf(q)), "tcpxb_norm_rope_forward");
  return {qOut, kOut};
}

std::tuple<Tensor, Tensor, Maybe, Maybe> normRopeBackward(Tensor dqOut, Tensor dkOut, Tensor q, Tensor k, Tensor cos, Tensor sin, Maybe wq, Maybe wk, double eps,
                                                          Maybe positions) {
  tcpxbNormRope a = checkNormRope(q, k, cos, sin, wq, wk, eps, positions);
  for (const auto& [name, t, x] : {std::tuple<const char*, const Tensor&, const Tensor&>{"dq_out", dqOut, q}, {"dk_out", dkOut, k}}) {
    TORCH_CHECK_VALUE(t.sizes() == x.sizes(), name, " has to be ", x.sizes(), ", got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " has to be ", x.scalar_type(), ", got ", t.scalar_type());
  }
  std::optional<c10::cuda::CUDAGuard> guard;
  const Maybe mq = q, mk = k, mcos = cos, msin = sin, mdq = dqOut, mdk = dkOut;
  noTangent({&mq, &mk, &mcos, &msin, &mdq, &mdk, &wq, &wk});
  onDevice(guard, q, {&mk, &mcos, &msin, &mdq, &mdk, &wq, &wk, &positions});
  Tensor dq = make(q, q.sizes()), dk = make(k, k.sizes()), partial;
  Maybe dwq, dwk;
  describe(a, cos, sin, wq, wk, positions);
  if (wq) {
    dwq = make(q, {a.d}), dwk = make(q, {a.d});
    partial = make(cos, {int64_t(tcpxb_norm_rope_scratch_bytes(a.d) / sizeof(float))});
    a.dwq = dwq->data_ptr(), a.dwk = dwk->data_ptr(), a.partial = partial.data_ptr<float>();
    a.q = heads(q), a.k = heads(k);
  }
  a.dq_out = heads(dqOut), a.dk_out = heads(dkOut);
  a.dq = dq.data_ptr(), a.dk = dk.data_ptr();
  done(tcpxb_norm_rope_backward(&a, streamOf(dq)), "tcpxb_norm_rope_backward");
  return {dq, dk, dwq, dwk};
}

// ------------------------------------------------------------------ AdamW
using List = std::vector<Tensor>;

// A list's tensors are contiguous, of one type, on one device, and as large as they have to be.
template <class Size> void checkList(const char* name, const List& ts, size_t count, ScalarType type, const Tensor& like, Size size) {
  TORCH_CHECK_VALUE(ts.size() == count, count, " tensors, but ", ts.size(), " ", name);
  for (size_t i = 0; i < count; i++) {
    const Tensor& t = ts[i];
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, "[", i, "] has to be ", type, ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.numel() == size(i), name, "[", i, "] has ", t.numel(), " elements, not ", size(i));
    TORCH_CHECK_VALUE(t.is_contiguous(), name, "[", i, "] has to be contiguous");
    TORCH_CHECK_VALUE(t.device() == like.device(), name, "[", i, "] is on ", t.device(), ", not on ", like.device());
  }
}

// The memory of a call's tensors.  What is written may not share a byte with anything else: two blocks would
// write the same elements, or read what another one has written, in an order that nothing gives.
class Ranges {
 public:
  void reserve(size_t n) { all_.reserve(n); }
  void* add(const Tensor& t, bool written) {
    void* p = t.data_ptr();
    const auto at = reinterpret_cast<uintptr_t>(p);
    if (t.numel()) all_.push_back({at, at + t.nbytes(), written});
    return p;
  }
  bool apart() {
    std::sort(all_.begin(), all_.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t read = 0, write = 0;  // ends so far
    for (const Range& r : all_) {
      if (r.begin < (r.written ? std::max(read, write) : write)) return false;
      uintptr_t& end = r.written ? write : read;
      end = std::max(end, r.end);
    }
    return true;
  }

 private:
  struct Range {
    uintptr_t begin, end;
    bool written;
  };
  std::vector<Range> all_;
};

Tensor gradNorm(const List& grads) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  const auto type = grads[0].scalar_type();
  TORCH_CHECK_TYPE(codeOf(type), "gradients have to be bfloat16, float16 or float32, got ", type);
  checkList("grads", grads, grads.size(), type, grads[0], [&](size_t i) { return grads[i].numel(); });
  std::optional<c10::cuda::CUDAGuard> guard;
  onDevice(guard, grads[0], {});
  std::vector<tcpxbAdamwTensor> table(grads.size());
  for (size_t i = 0; i < grads.size(); i++) table[i].g = grads[i].data_ptr(), table[i].n = grads[i].numel();
  const int count = int(grads.size());
  Tensor norm = make(grads[0], {}, at::kFloat), scratch = make(grads[0], {int64_t(tcpxb_grad_norm_scratch_bytes(table.data(), count))}, at::kByte);
  done(tcpxb_grad_norm(table.data(), count, codeOf(type), grads[0].get_device(), norm.data_ptr<float>(), scratch.data_ptr(), streamOf(norm)), "tcpxb_grad_norm");
  return norm;
}

Maybe adamwStep(const List& params, const List& grads, const List& ms, const List& vs, const std::variant<Tensor, List>& steps, double lr, double beta1, double beta2, double eps,
                double decay, std::optional<double> maxNorm, Maybe norm, std::optional<List> mScales, std::optional<List> vScales, std::optional<List> masters) {
  TORCH_CHECK_VALUE(!params.empty(), "no tensors");
  const Tensor& first = params[0];
  const auto type = first.scalar_type();
  TORCH_CHECK_TYPE(codeOf(type), "params have to be bfloat16, float16 or float32, got ", type);
  TORCH_CHECK_VALUE(mScales.has_value() == vScales.has_value(), "8-bit states need the scales of both");
  const size_t count = params.size();
  const auto size = [&](size_t i) { return params[i].numel(); };
  const auto state = mScales ? at::kFloat8_e4m3fn : at::kFloat;
  checkList("params", params, count, type, first, size);
  checkList("grads", grads, count, type, first, size);
  checkList("exp_avgs", ms, count, state, first, size);
  checkList("exp_avg_sqs", vs, count, state, first, size);
  if (mScales) {
    const auto blocks = [&](size_t i) { return (params[i].numel() + TCPXB_ADAMW_BLOCK - 1) / TCPXB_ADAMW_BLOCK; };
    checkList("exp_avg_scales", *mScales, count, at::kFloat, first, blocks);
    checkList("exp_avg_sq_scales", *vScales, count, at::kFloat, first, blocks);
  }
  if (masters) {
    TORCH_CHECK_VALUE(type != at::kFloat, "masters stand behind 16-bit params");
    checkList("masters", *masters, count, at::kFloat, first, size);
  }
  std::vector<tcpxbAdamwTensor> table(count);
  Ranges ranges;
  ranges.reserve(count * 8 + 2);
  const auto write = [&](const Tensor& t) { return ranges.add(t, true); };
  if (const auto* whole = std::get_if<Tensor>(&steps)) {
    const Tensor& t = *whole;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, "steps has to be int32, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.dim() == 1 && size_t(t.size(0)) == count && t.is_contiguous() && t.device() == first.device(), "steps has to be a contiguous [", count,
                      "] on the same device, got ", t.sizes());
    auto* first = static_cast<int32_t*>(write(t));
    for (size_t i = 0; i < count; i++) table[i].step = first + i;
  } else {
    const List& list = std::get<List>(steps);
    checkList("steps", list, count, at::kInt, first, [](size_t) { return 1; });
    for (size_t i = 0; i < count; i++) table[i].step = static_cast<int32_t*>(write(list[i]));
  }
  for (size_t i = 0; i < count; i++) {
    table[i].p = write(params[i]), table[i].g = ranges.add(grads[i], false), table[i].m = write(ms[i]), table[i].v = write(vs[i]), table[i].n = params[i].numel();
    if (mScales) table[i].m_scale = static_cast<float*>(write((*mScales)[i])), table[i].v_scale = static_cast<float*>(write((*vScales)[i]));
    if (masters) table[i].master = static_cast<float*>(write((*masters)[i]));
  }
  if (norm) ranges.add(*norm, false);
  TORCH_CHECK_VALUE(ranges.apart(), "a tensor that is written is given twice, or shares memory with another one");
  const auto good = [](double x) { return x >= 0 && x < INFINITY; };
  TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && good(eps) && good(lr) && good(decay), "bad numbers: lr ", lr, ", betas (", beta1, ", ",
                    beta2, "), eps ", eps, ", weight_decay ", decay);
  TORCH_CHECK_VALUE(!maxNorm || good(*maxNorm), "max_grad_norm has to be finite and not below zero");
  TORCH_CHECK_VALUE(!norm || (norm->scalar_type() == at::kFloat && norm->numel() == 1 && maxNorm), "norm has to be one float32 value, given with max_grad_norm");
  std::optional<c10::cuda::CUDAGuard> guard;
  onDevice(guard, first, {&norm});
  tcpxbAdamw a = {};
  a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.eps = eps, a.weight_decay = decay;
  a.compute_norm = maxNorm && !norm;
  if (a.compute_norm) norm = make(first, {}, at::kFloat);
  if (maxNorm) a.grad_norm = norm->data_ptr<float>(), a.max_norm = float(*maxNorm);
  a.state_bits = mScales ? 8 : 32, a.dtype = codeOf(type), a.device = first.get_device();
  Tensor scratch = make(first, {int64_t(tcpxb_adamw_scratch_bytes(table.data(), int(count)))}, at::kByte);
  a.scratch = scratch.data_ptr();
  done(tcpxb_adamw_step(table.data(), int(count), &a, streamOf(first)), "tcpxb_adamw_step");
  for (const Tensor& p : params)
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();  // autograd learns of the update, as of any other in place
  return norm;
}

// Other Python threads run meanwhile: an allocation or a launch may wait for the device, and what the
// device waits for may be another thread's to give.
struct Release {
  PyThreadState* state = PyEval_SaveThread();
  ~Release() { PyEval_RestoreThread(state); }
};

}  // namespace

PYBIND11_MODULE(tcpxb_train_torch, m) {
  using Unlocked = py::call_guard<Release>;
  m.def("attention_forward", &attentionForward, Unlocked());
  m.def("attention_backward", &attentionBackward, Unlocked());
  m.def("norm_rope_forward", &normRopeForward, Unlocked());
  m.def("norm_rope_backward", &normRopeBackward, Unlocked());
  m.def("grad_norm", &gradNorm, Unlocked());
  m.def("adamw_step", &adamwStep, Unlocked());
}
