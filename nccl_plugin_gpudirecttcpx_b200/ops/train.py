"""Python bindings of the training step's sm_100a operators.

`attention`, `qk_norm_rope` and `adamw_step` (with `grad_norm` and the optimizer `AdamW` on
top) are what a decoder's training step needs next to its gradient collectives.  Each takes
torch CUDA tensors, passes raw pointers and the device's current stream to the C ABI in
`csrc/include/tcpxb/train.h`, and raises if the native library is missing: there is no eager
fallback.  Arguments are checked on the host before anything is queued: a wrong shape, size or
option is a `ValueError`, a wrong type a `TypeError`.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from ..utils import native

STATE_BLOCK = 256  # elements that share a scale of an 8-bit AdamW state
MAX_HEAD_SIZE = 128  # of attention
MAX_NORM_HEAD_SIZE = 256  # of qk_norm_rope

_CODES = {torch.bfloat16: 1, torch.float32: 2, torch.float16: 3}
_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class _Heads(ctypes.Structure):
    _fields_ = [("ptr", _vp), ("stride_b", _i64), ("stride_s", _i64), ("stride_h", _i64)]


class _Attention(ctypes.Structure):
    _fields_ = [("q", _Heads), ("k", _Heads), ("v", _Heads), ("out", _vp), ("lse", _vp), ("dout", _Heads), ("dq", _vp), ("dk", _vp),
                ("dv", _vp), ("delta", _vp), ("key_lengths", _vp), ("b", _i32), ("sq", _i32), ("sk", _i32), ("heads", _i32),
                ("kv_heads", _i32), ("d", _i32), ("scale", _f32), ("causal", _i32), ("dtype", _i32), ("status", _vp)]


class _NormRope(ctypes.Structure):
    _fields_ = [("q", _Heads), ("k", _Heads), ("wq", _vp), ("wk", _vp), ("cos", _vp), ("sin", _vp), ("pos", _vp), ("q_out", _vp),
                ("k_out", _vp), ("dq_out", _Heads), ("dk_out", _Heads), ("dq", _vp), ("dk", _vp), ("dwq", _vp), ("dwk", _vp),
                ("partial", _vp), ("b", _i32), ("s", _i32), ("heads", _i32), ("kv_heads", _i32), ("d", _i32), ("positions", _i32),
                ("eps", _f32), ("dtype", _i32)]


class _AdamwTensor(ctypes.Structure):
    _fields_ = [("p", _vp), ("g", _vp), ("m", _vp), ("v", _vp), ("m_scale", _vp), ("v_scale", _vp), ("master", _vp), ("step", _vp),
                ("n", _i64)]


class _Adamw(ctypes.Structure):
    _fields_ = [("lr", _f32), ("beta1", _f32), ("beta2", _f32), ("eps", _f32), ("weight_decay", _f32), ("grad_norm", _vp),
                ("max_norm", _f32), ("state_bits", _i32), ("dtype", _i32), ("scratch", _vp)]


_lib = None


def _t():
    global _lib
    if _lib is None:
        lib = native.load("libtcpxb_train.so")
        lib.tcpxb_train_last_error.restype = ctypes.c_char_p
        for name in ("tcpxb_attention_forward", "tcpxb_attention_backward", "tcpxb_norm_rope_forward", "tcpxb_norm_rope_backward"):
            getattr(lib, name).argtypes = [_vp, _vp]
        lib.tcpxb_norm_rope_scratch_bytes.restype = ctypes.c_size_t
        lib.tcpxb_adamw_scratch_bytes.restype = ctypes.c_size_t
        lib.tcpxb_adamw_step.argtypes = [_vp, ctypes.c_int, _vp, _vp]
        lib.tcpxb_grad_norm_scratch_bytes.argtypes = [_vp, ctypes.c_int]
        lib.tcpxb_grad_norm_scratch_bytes.restype = ctypes.c_size_t
        lib.tcpxb_grad_norm.argtypes = [_vp, ctypes.c_int, ctypes.c_int, _vp, _vp, _vp]
        _lib = lib
    return _lib


def _call(name: str, device: torch.device, *args) -> None:
    """Runs a C entry on the tensors' device, whichever is current, and on that device's current stream."""
    with torch.cuda.device(device):
        rc = getattr(_t(), name)(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {_t().tcpxb_train_last_error().decode()}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _on_one_device(*ts: Optional[torch.Tensor]) -> torch.device:
    devices = {t.device for t in ts if t is not None}
    if len(devices) != 1 or next(iter(devices)).type != "cuda":
        raise ValueError(f"all tensors have to be on one CUDA device, got {sorted(map(str, devices))}")
    return next(iter(devices))


def _heads(t: torch.Tensor) -> tuple:
    """(descriptor, tensor that it points into): the tensor itself where its head rows start on 16-byte
    boundaries and are not broadcast, else a contiguous copy."""
    size = t.element_size()
    strides = [st if n > 1 else 16 for n, st in zip(t.shape, t.stride())]
    if (t.shape[3] > 1 and t.stride(3) != 1) or t.data_ptr() % 16 or any(st * size % 16 or st == 0 for st in strides[:3]):
        t = t.clone(memory_format=torch.contiguous_format)
        strides = list(t.stride())
    return _Heads(t.data_ptr(), *strides[:3]), t


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------- attention
def _check_attention(q, k, v, scale, key_lengths) -> float:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} has to be [batch, tokens, heads, head size], got {tuple(t.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"attention takes bfloat16 or float16 of one kind, got {q.dtype}, {k.dtype}, {v.dtype}")
    b, _, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if h < 1 or k.shape[2] < 1 or h % k.shape[2]:
        raise ValueError(f"{h} query heads are no multiple of {k.shape[2]} key heads")
    if d % 8 or not 8 <= d <= MAX_HEAD_SIZE:
        raise ValueError(f"the head size has to be a multiple of 8 up to {MAX_HEAD_SIZE}, got {d}")
    if key_lengths is not None:
        if key_lengths.dtype != torch.int32:
            raise TypeError(f"key_lengths has to be int32, got {key_lengths.dtype}")
        if key_lengths.shape != (b,):
            raise ValueError(f"key_lengths has to be [{b}], got {tuple(key_lengths.shape)}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < 1e30:
        raise ValueError(f"scale has to be finite and above zero, got {scale}")
    return scale


def _attention_args(q, k, v, scale, causal, key_lengths):
    a = _Attention()
    a.q, q = _heads(q)
    a.k, k = _heads(k)
    a.v, v = _heads(v)
    key_lengths = None if key_lengths is None else key_lengths.contiguous()
    a.key_lengths = _ptr(key_lengths)
    a.b, a.sq, a.heads, a.d = q.shape
    a.sk, a.kv_heads = k.shape[1:3]
    a.scale, a.causal, a.dtype = scale, int(bool(causal)), _CODES[q.dtype]
    return a, (q, k, v, key_lengths)


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: Optional[float] = None,
                      key_lengths: Optional[torch.Tensor] = None) -> tuple:
    """(out, lse) of softmax(scale q k^T) v; not recorded by autograd (see `attention`).

    q is [batch, queries, heads, head size], k and v [batch, keys, key heads, head size]; query heads
    are a multiple of the key heads (head h reads key head h // (heads // key heads)).  bfloat16 or
    float16, head size a multiple of 8 up to 128.  Any strides: tensors whose head rows do not start on
    16-byte boundaries are copied first.  `causal`: query i sees keys up to i + keys - queries.
    `key_lengths` ([batch], int32): keys at and behind a batch's length are not seen, whatever they
    hold.  A query that sees no key gets zeros.  `out` is contiguous; `lse` [batch, heads, queries]
    (float32) is the natural logarithm of each row's sum of exponentials, -inf for an empty row."""
    scale = _check_attention(q, k, v, scale, key_lengths)
    dev = _on_one_device(q, k, v, key_lengths)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=dev)
    a, keep = _attention_args(q, k, v, scale, causal, key_lengths)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    _call("tcpxb_attention_forward", dev, ctypes.byref(a))
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, *,
                       causal: bool = False, scale: Optional[float] = None, key_lengths: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dv) from what `attention_forward` returned for the same arguments.  The probabilities
    are computed again from the scores and `lse`.  The same inputs give the same bits every time."""
    scale = _check_attention(q, k, v, scale, key_lengths)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape:
            raise ValueError(f"{name} has to be {tuple(q.shape)}, got {tuple(t.shape)}")
        if t.dtype != q.dtype:
            raise TypeError(f"{name} has to be {q.dtype}, got {t.dtype}")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]):
        raise ValueError(f"lse has to be [batch, heads, queries], got {tuple(lse.shape)}")
    if lse.dtype != torch.float32:
        raise TypeError(f"lse has to be float32, got {lse.dtype}")
    dev = _on_one_device(dout, q, k, v, out, lse, key_lengths)
    a, keep = _attention_args(q, k, v, scale, causal, key_lengths)
    a.dout, dout = _heads(dout)
    out, lse = _aligned(out), lse.contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    delta = torch.empty_like(lse)
    a.out, a.lse, a.delta = out.data_ptr(), lse.data_ptr(), delta.data_ptr()
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    _call("tcpxb_attention_backward", dev, ctypes.byref(a))
    return dq, dk, dv


class _AttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale, key_lengths):
        out, lse = attention_forward(q, k, v, causal=causal, scale=scale, key_lengths=key_lengths)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths)
        ctx.how = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_lengths = ctx.saved_tensors
        causal, scale = ctx.how
        return (*attention_backward(dout, q, k, v, out, lse, causal=causal, scale=scale, key_lengths=key_lengths), None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: Optional[float] = None,
              key_lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`attention_forward`'s `out`, differentiable in q, k and v (once)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFunction.apply(q, k, v, causal, scale, key_lengths)
    return attention_forward(q, k, v, causal=causal, scale=scale, key_lengths=key_lengths)[0]


# ---------------------------------------------------------------- qk_norm_rope
def _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions) -> None:
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 4:
            raise ValueError(f"{name} has to be [batch, tokens, heads, head size], got {tuple(t.shape)}")
    if q.dtype not in _CODES or k.dtype != q.dtype:
        raise TypeError(f"q and k have to be bfloat16, float16 or float32 of one kind, got {q.dtype} and {k.dtype}")
    b, s, h, d = q.shape
    if k.shape[:2] != q.shape[:2] or k.shape[3] != d or h < 1 or k.shape[2] < 1:
        raise ValueError(f"shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}")
    if d % 8 or not 8 <= d <= MAX_NORM_HEAD_SIZE:
        raise ValueError(f"the head size has to be a multiple of 8 up to {MAX_NORM_HEAD_SIZE}, got {d}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError(f"cos and sin have to be float32, got {cos.dtype} and {sin.dtype}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != d // 2:
        raise ValueError(f"cos and sin have to be [positions, {d // 2}], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if positions is None:
        if cos.shape[0] < s:
            raise ValueError(f"the tables hold {cos.shape[0]} positions of {s}")
    else:
        if positions.dtype != torch.int64:
            raise TypeError(f"positions has to be int64, got {positions.dtype}")
        if positions.shape != (b, s):
            raise ValueError(f"positions has to be [{b}, {s}], got {tuple(positions.shape)}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight come together")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name} has to be [{d}], got {tuple(w.shape)}")
        if w is not None and w.dtype != q.dtype:
            raise TypeError(f"{name} has to be {q.dtype}, got {w.dtype}")
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps has to be finite and not below zero, got {eps}")


def _norm_rope_args(q, k, cos, sin, q_weight, k_weight, eps, positions):
    a = _NormRope()
    cos, sin, q_weight, k_weight = _aligned(cos), _aligned(sin), _aligned(q_weight), _aligned(k_weight)
    positions = None if positions is None else positions.contiguous()
    a.cos, a.sin, a.wq, a.wk, a.pos = _ptr(cos), _ptr(sin), _ptr(q_weight), _ptr(k_weight), _ptr(positions)
    a.b, a.s, a.heads, a.d = q.shape
    a.kv_heads, a.positions, a.eps, a.dtype = k.shape[2], cos.shape[0], eps, _CODES[q.dtype]
    return a, (cos, sin, q_weight, k_weight, positions)


def _norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions) -> tuple:
    _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions)
    dev = _on_one_device(q, k, cos, sin, q_weight, k_weight, positions)
    a, keep = _norm_rope_args(q, k, cos, sin, q_weight, k_weight, eps, positions)
    a.q, q = _heads(q)
    a.k, k = _heads(k)
    q_out, k_out = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    _call("tcpxb_norm_rope_forward", dev, ctypes.byref(a))
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          eps: float = 1e-6, positions: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dq_weight, dk_weight) of `qk_norm_rope` from the gradients of its outputs and its own
    arguments (the weights' are None without weights).  The same inputs give the same bits every time."""
    _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions)
    for name, t, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if t.shape != x.shape:
            raise ValueError(f"{name} has to be {tuple(x.shape)}, got {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} has to be {x.dtype}, got {t.dtype}")
    dev = _on_one_device(dq_out, dk_out, q, k, cos, sin, q_weight, k_weight, positions)
    a, keep = _norm_rope_args(q, k, cos, sin, q_weight, k_weight, eps, positions)
    a.dq_out, dq_out = _heads(dq_out)
    a.dk_out, dk_out = _heads(dk_out)
    dq, dk = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
    a.dq, a.dk = dq.data_ptr(), dk.data_ptr()
    dwq = dwk = None
    if q_weight is not None:
        a.q, q = _heads(q)
        a.k, k = _heads(k)
        dwq, dwk = torch.empty_like(q_weight), torch.empty_like(k_weight)
        partial = torch.empty(_t().tcpxb_norm_rope_scratch_bytes(a.d), dtype=torch.uint8, device=dev)
        a.dwq, a.dwk, a.partial = dwq.data_ptr(), dwk.data_ptr(), partial.data_ptr()
    _call("tcpxb_norm_rope_backward", dev, ctypes.byref(a))
    return dq, dk, dwq, dwk


class _NormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, q_weight, k_weight, eps, positions):
        out = _norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions)
        normed = q_weight is not None
        # the rotation alone is turned back without its inputs
        ctx.save_for_backward(q if normed else None, k if normed else None, cos, sin, q_weight, k_weight, positions)
        ctx.eps = eps
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, cos, sin, q_weight, k_weight, positions = ctx.saved_tensors
        grads = qk_norm_rope_backward(dq_out, dk_out, dq_out if q is None else q, dk_out if k is None else k, cos, sin, q_weight, k_weight,
                                      eps=ctx.eps, positions=positions)
        return (*grads[:2], None, None, *grads[2:], None, None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6, positions: Optional[torch.Tensor] = None) -> tuple:
    """Queries and keys, each head normalised by its root mean square and scaled by a weight, then rotated
    by its token's position; differentiable (once) in q, k and the weights, not in the tables.

    q is [batch, tokens, heads, head size], k the same with its own number of heads; bfloat16, float16 or
    float32, head size a multiple of 8 up to 256, any strides.  `cos` and `sin` ([positions, head size / 2],
    float32) turn the pairs (x[2i], x[2i + 1]); token t of a batch takes row t, or row `positions[b, t]`
    (int64).  A position outside the tables gives NaN.  Without weights there is no norm.  All in 32 bits,
    rounded once; outputs are contiguous."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _NormRopeFunction.apply(q, k, cos, sin, q_weight, k_weight, eps, positions)
    return _norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions)


# ----------------------------------------------------------------------- AdamW
def _flat_list(name: str, ts: Sequence[torch.Tensor], like: Sequence[torch.Tensor], dtype: torch.dtype, numels=None) -> None:
    if len(ts) != len(like):
        raise ValueError(f"{len(like)} tensors, but {len(ts)} {name}")
    for i, (t, p) in enumerate(zip(ts, like)):
        if t.dtype != dtype:
            raise TypeError(f"{name}[{i}] has to be {dtype}, got {t.dtype}")
        if t.numel() != (p.numel() if numels is None else numels[i]):
            raise ValueError(f"{name}[{i}] has {t.numel()} elements")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}] has to be contiguous")


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """Root of the sum of all squares, as a float32 scalar on the device.  Contiguous CUDA tensors of one
    type (bfloat16, float16, float32); squares of a few elements are added in 32 bits, those sums in 64,
    in an order that depends on the sizes alone."""
    grads = list(grads)
    if not grads:
        raise ValueError("no gradients")
    if grads[0].dtype not in _CODES:
        raise TypeError(f"gradients have to be bfloat16, float16 or float32, got {grads[0].dtype}")
    _flat_list("grads", grads, grads, grads[0].dtype)
    dev = _on_one_device(*grads)
    table = (_AdamwTensor * len(grads))()
    for e, g in zip(table, grads):
        e.g, e.n = g.data_ptr(), g.numel()
    return _queue_norm(table, len(grads), grads[0].dtype, dev)


def _queue_norm(table, count: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    norm = torch.empty((), dtype=torch.float32, device=dev)
    scratch = torch.empty(_t().tcpxb_grad_norm_scratch_bytes(table, count), dtype=torch.uint8, device=dev)
    _call("tcpxb_grad_norm", dev, table, count, _CODES[dtype], norm.data_ptr(), scratch.data_ptr())
    return norm


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: torch.Tensor, *, lr: float, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, max_grad_norm: Optional[float] = None, norm: Optional[torch.Tensor] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
               masters: Optional[Sequence[torch.Tensor]] = None) -> Optional[torch.Tensor]:
    """One AdamW step over all tensors, in place, in two launches (four with clipping).

    `params` and `grads`: contiguous tensors of one type (bfloat16, float16, float32) on one device.
    States in 32 bits: `exp_avgs` and `exp_avg_sqs` are float32 tensors of the params' sizes.  In 8 bits:
    float8_e4m3fn tensors with `exp_avg_scales` and `exp_avg_sq_scales`, one float32 per 256 elements; a
    state's value is code times scale, and `exp_avg_sqs` holds the root.  `steps` ([number of tensors],
    int32) counts each tensor's updates and is advanced.  `max_grad_norm`: gradients are scaled by
    min(1, max_grad_norm / (norm + 1e-6)), where `norm` is theirs over all tensors (computed here and
    returned), or the given float32 device scalar, for lists that share one.  `masters`: float32 weights
    that are updated and rounded into 16-bit `params`.  Nothing is copied to or from the host: the call can
    be captured into a graph, which then keeps the given numbers and pointers."""
    params, grads, exp_avgs, exp_avg_sqs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    if not params:
        raise ValueError("no tensors")
    dtype = params[0].dtype
    if dtype not in _CODES:
        raise TypeError(f"params have to be bfloat16, float16 or float32, got {dtype}")
    bits = 8 if exp_avg_scales is not None else 32
    if (exp_avg_sq_scales is None) != (bits == 32):
        raise ValueError("8-bit states need the scales of both")
    _flat_list("params", params, params, dtype)
    _flat_list("grads", grads, params, dtype)
    state = torch.float8_e4m3fn if bits == 8 else torch.float32
    _flat_list("exp_avgs", exp_avgs, params, state)
    _flat_list("exp_avg_sqs", exp_avg_sqs, params, state)
    lists = [params, grads, exp_avgs, exp_avg_sqs]
    if bits == 8:
        exp_avg_scales, exp_avg_sq_scales = list(exp_avg_scales), list(exp_avg_sq_scales)
        blocks = [-(-p.numel() // STATE_BLOCK) for p in params]
        _flat_list("exp_avg_scales", exp_avg_scales, params, torch.float32, blocks)
        _flat_list("exp_avg_sq_scales", exp_avg_sq_scales, params, torch.float32, blocks)
        lists += [exp_avg_scales, exp_avg_sq_scales]
    if masters is not None:
        masters = list(masters)
        if dtype == torch.float32:
            raise ValueError("masters stand behind 16-bit params")
        _flat_list("masters", masters, params, torch.float32)
        lists.append(masters)
    if steps.dtype != torch.int32:
        raise TypeError(f"steps has to be int32, got {steps.dtype}")
    if steps.shape != (len(params),) or not steps.is_contiguous():
        raise ValueError(f"steps has to be a contiguous [{len(params)}], got {tuple(steps.shape)}")
    written = [t.data_ptr() for ts in lists if ts is not grads for t in ts if t.numel()]
    if len(set(written)) != len(written):
        raise ValueError("a tensor is given twice")
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and 0 <= eps < math.inf and 0 <= lr < math.inf and 0 <= weight_decay < math.inf):
        raise ValueError(f"bad numbers: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
    if max_grad_norm is not None and not 0 <= max_grad_norm < math.inf:
        raise ValueError(f"max_grad_norm has to be finite and not below zero, got {max_grad_norm}")
    if norm is not None and (norm.dtype != torch.float32 or norm.numel() != 1 or max_grad_norm is None):
        raise ValueError("norm has to be one float32 value, given with max_grad_norm")
    dev = _on_one_device(steps, norm, *(t for ts in lists for t in ts))
    count = len(params)
    table = (_AdamwTensor * count)()
    step_ptr = steps.data_ptr()
    for i, e in enumerate(table):
        e.p, e.g, e.m, e.v = params[i].data_ptr(), grads[i].data_ptr(), exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr()
        e.step, e.n = step_ptr + 4 * i, params[i].numel()
        if bits == 8:
            e.m_scale, e.v_scale = exp_avg_scales[i].data_ptr(), exp_avg_sq_scales[i].data_ptr()
        if masters is not None:
            e.master = masters[i].data_ptr()
    if max_grad_norm is not None and norm is None:
        norm = _queue_norm(table, count, dtype, dev)
    scratch = torch.empty(_t().tcpxb_adamw_scratch_bytes(count), dtype=torch.uint8, device=dev)
    a = _Adamw(lr, beta1, beta2, eps, weight_decay, _ptr(norm), max_grad_norm or 0.0, bits, _CODES[dtype], scratch.data_ptr())
    _call("tcpxb_adamw_step", dev, table, count, ctypes.byref(a))
    return norm
