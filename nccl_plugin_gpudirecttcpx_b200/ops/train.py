"""Python bindings of the training step's sm_100a operators.

`attention`, `qk_norm_rope` and `adamw_step` (with `grad_norm` and the optimizer `AdamW` on
top) are what a decoder's training step needs next to its gradient collectives.  Each takes
torch CUDA tensors, passes raw pointers and the device's current stream to the C ABI in
`csrc/include/tcpxb/train.h`, and raises if the native library is missing: there is no eager
fallback.  Arguments are checked on the host before anything is queued: a wrong shape, size or
option is a `ValueError`, a wrong type a `TypeError`.
"""
from __future__ import annotations

import array
import ctypes
import itertools
import math
import operator
import struct
from typing import Optional, Sequence

import torch

from ..utils import native

STATE_BLOCK = 256  # elements that share a scale of an 8-bit AdamW state
MAX_HEAD_SIZE = 128  # of attention
MAX_NORM_HEAD_SIZE = 256  # of qk_norm_rope

_CODES = {torch.bfloat16: 1, torch.float32: 2, torch.float16: 3}
_vp = ctypes.c_void_p


# The C entries' argument structs (csrc/include/tcpxb/train.h); a heads descriptor is 4q.
_ATTENTION = struct.Struct("@12q2P4q5P6if2iP")
_NORM_ROPE = struct.Struct("@8q7P8q5P6ifi")
_ADAMW = struct.Struct("@5dPf3iP")


_entries: dict = {}


def _t():
    return native.load("libtcpxb_train.so")


def _entry(name: str):
    """A C entry with its signature."""
    if not _entries:
        lib = _t()
        size, text, i32 = ctypes.c_size_t, ctypes.c_char_p, ctypes.c_int
        for entry, result, *args in (
                ("tcpxb_train_last_error", text),
                ("tcpxb_attention_forward", i32, _vp, _vp), ("tcpxb_attention_backward", i32, _vp, _vp),
                ("tcpxb_norm_rope_forward", i32, _vp, _vp), ("tcpxb_norm_rope_backward", i32, _vp, _vp), ("tcpxb_norm_rope_scratch_bytes", size, i32),
                ("tcpxb_adamw_scratch_bytes", size, _vp, i32), ("tcpxb_adamw_step", i32, _vp, i32, _vp, _vp),
                ("tcpxb_grad_norm_scratch_bytes", size, _vp, i32), ("tcpxb_grad_norm", i32, _vp, i32, i32, _vp, _vp, _vp)):
            f = getattr(lib, entry)
            f.restype, f.argtypes = result, args
            _entries[entry] = f
    return _entries[name]


def _call(name: str, device: int, *args) -> None:
    """Runs a C entry on the tensors' device, whichever is current, and on that device's current stream."""
    entry = _entries.get(name) or _entry(name)
    if torch._C._cuda_getDevice() == device:
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {_entry('tcpxb_train_last_error')().decode()}")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _on_one_device(first: torch.Tensor, *rest: Optional[torch.Tensor]) -> int:
    """The number of the CUDA device that all of them are on."""
    device = first.get_device()
    if device >= 0 and first.is_cuda:
        for t in rest:
            if t is not None and t.get_device() != device:
                break
        else:
            return device
    raise ValueError(f"all tensors have to be on one CUDA device, got {sorted({str(t.device) for t in (first, *rest) if t is not None})}")


def _heads(t: torch.Tensor, per: int) -> tuple:
    """(tensor, pointer, strides of batch, token and head): of the tensor itself where its head rows start on
    16-byte boundaries (`per` elements) and are not broadcast, else of a contiguous copy."""
    b, s, h, d = t.shape
    sb, ss, sh, sd = t.stride()
    # the stride of a single entry is of no influence
    if b == 1:
        sb = 16
    if s == 1:
        ss = 16
    if h == 1:
        sh = 16
    p = t.data_ptr()
    if p % 16 or (sb | ss | sh) % per or (sd != 1 and d > 1) or not (sb and ss and sh):
        t = t.clone(memory_format=torch.contiguous_format)
        sb, ss, sh = t.stride()[:3]
        p = t.data_ptr()
    return t, p, sb, ss, sh


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------- attention
def _check_attention(q, k, v, scale, key_lengths) -> tuple:
    """(batch, queries, keys, heads, key heads, head size, scale)."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v have to be [batch, tokens, heads, head size], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    dtype = q.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError(f"attention takes bfloat16 or float16 of one kind, got {dtype}, {k.dtype}, {v.dtype}")
    b, sq, h, d = q.shape
    kb, sk, hk, kd = k.shape
    if kb != b or kd != d or v.shape != k.shape:
        raise ValueError(f"shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"{h} query heads are no multiple of {hk} key heads")
    if d % 8 or not 8 <= d <= MAX_HEAD_SIZE:
        raise ValueError(f"the head size has to be a multiple of 8 up to {MAX_HEAD_SIZE}, got {d}")
    if key_lengths is not None:
        if key_lengths.dtype is not torch.int32:
            raise TypeError(f"key_lengths has to be int32, got {key_lengths.dtype}")
        if key_lengths.shape != (b,):
            raise ValueError(f"key_lengths has to be [{b}], got {tuple(key_lengths.shape)}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < 1e30:
        raise ValueError(f"scale has to be finite and above zero, got {scale}")
    return b, sq, sk, h, hk, d, scale


def _check_status(status: Optional[torch.Tensor]) -> None:
    if status is not None and (status.dtype is not torch.int32 or status.numel() < 1 or not status.is_contiguous()):
        raise ValueError("status has to be a contiguous int32 tensor (ops.status_buffer())")


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: Optional[float] = None,
                      key_lengths: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> tuple:
    """(out, lse) of softmax(scale q k^T) v; not recorded by autograd (see `attention`).

    q is [batch, queries, heads, head size], k and v [batch, keys, key heads, head size]; query heads
    are a multiple of the key heads (head h reads key head h // (heads // key heads)).  bfloat16 or
    float16, head size a multiple of 8 up to 128.  Any strides: tensors whose head rows do not start on
    16-byte boundaries are copied first.  `causal`: query i sees keys up to i + keys - queries.
    `key_lengths` ([batch], int32): keys at and behind a batch's length are not seen, whatever they
    hold.  A query that sees no key gets zeros.  `out` is contiguous; `lse` [batch, heads, queries]
    (float32) is the natural logarithm of each row's sum of exponentials, -inf for an empty row.
    `status` (`ops.status_buffer()`): its first word becomes 3 where a wait inside the kernel ran out of
    time and the outputs are void."""
    b, sq, sk, h, hk, d, scale = _check_attention(q, k, v, scale, key_lengths)
    _check_status(status)
    dev = _on_one_device(q, k, v, key_lengths, status)
    out, lse = q.new_empty((b, sq, h, d)), q.new_empty((b, h, sq), dtype=torch.float32)
    q, *qa = _heads(q, 8)
    k, *ka = _heads(k, 8)
    v, *va = _heads(v, 8)
    if key_lengths is not None:
        key_lengths = key_lengths.contiguous()
    _call("tcpxb_attention_forward", dev, _ATTENTION.pack(*qa, *ka, *va, out.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, _ptr(key_lengths),
                                                          b, sq, sk, h, hk, d, scale, bool(causal), _CODES[q.dtype], _ptr(status)))
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, *,
                       causal: bool = False, scale: Optional[float] = None, key_lengths: Optional[torch.Tensor] = None,
                       status: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dv) from what `attention_forward` returned for the same arguments.  The probabilities
    are computed again from the scores and `lse`.  The same inputs give the same bits every time."""
    b, sq, sk, h, hk, d, scale = _check_attention(q, k, v, scale, key_lengths)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape:
            raise ValueError(f"{name} has to be {tuple(q.shape)}, got {tuple(t.shape)}")
        if t.dtype is not q.dtype:
            raise TypeError(f"{name} has to be {q.dtype}, got {t.dtype}")
    if lse.shape != (b, h, sq):
        raise ValueError(f"lse has to be [batch, heads, queries], got {tuple(lse.shape)}")
    if lse.dtype is not torch.float32:
        raise TypeError(f"lse has to be float32, got {lse.dtype}")
    _check_status(status)
    dev = _on_one_device(dout, q, k, v, out, lse, key_lengths, status)
    dq, dk, dv = q.new_empty((b, sq, h, d)), k.new_empty((b, sk, hk, d)), v.new_empty((b, sk, hk, d))
    delta = lse.new_empty((b, h, sq))
    out, lse = _aligned(out), lse.contiguous()
    q, *qa = _heads(q, 8)
    k, *ka = _heads(k, 8)
    v, *va = _heads(v, 8)
    dout, *da = _heads(dout, 8)
    if key_lengths is not None:
        key_lengths = key_lengths.contiguous()
    _call("tcpxb_attention_backward", dev, _ATTENTION.pack(*qa, *ka, *va, out.data_ptr(), lse.data_ptr(), *da, dq.data_ptr(), dk.data_ptr(),
                                                           dv.data_ptr(), delta.data_ptr(), _ptr(key_lengths), b, sq, sk, h, hk, d, scale,
                                                           bool(causal), _CODES[q.dtype], _ptr(status)))
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
def _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions) -> tuple:
    """(batch, tokens, heads, key heads, head size, rows of the tables)."""
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k have to be [batch, tokens, heads, head size], got {tuple(q.shape)} and {tuple(k.shape)}")
    dtype = q.dtype
    if dtype not in _CODES or k.dtype is not dtype:
        raise TypeError(f"q and k have to be bfloat16, float16 or float32 of one kind, got {dtype} and {k.dtype}")
    b, s, h, d = q.shape
    kb, ks, hk, kd = k.shape
    if kb != b or ks != s or kd != d or h < 1 or hk < 1:
        raise ValueError(f"shapes do not match: q {tuple(q.shape)}, k {tuple(k.shape)}")
    if d % 8 or not 8 <= d <= MAX_NORM_HEAD_SIZE:
        raise ValueError(f"the head size has to be a multiple of 8 up to {MAX_NORM_HEAD_SIZE}, got {d}")
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise TypeError(f"cos and sin have to be float32, got {cos.dtype} and {sin.dtype}")
    table = cos.shape
    if len(table) != 2 or sin.shape != table or table[1] != d // 2:
        raise ValueError(f"cos and sin have to be [positions, {d // 2}], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if positions is None:
        if table[0] < s:
            raise ValueError(f"the tables hold {table[0]} positions of {s}")
    else:
        if positions.dtype is not torch.int64:
            raise TypeError(f"positions has to be int64, got {positions.dtype}")
        if positions.shape != (b, s):
            raise ValueError(f"positions has to be [{b}, {s}], got {tuple(positions.shape)}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight come together")
    if q_weight is not None:
        if q_weight.shape != (d,) or k_weight.shape != (d,):
            raise ValueError(f"the weights have to be [{d}], got {tuple(q_weight.shape)} and {tuple(k_weight.shape)}")
        if q_weight.dtype is not dtype or k_weight.dtype is not dtype:
            raise TypeError(f"the weights have to be {dtype}, got {q_weight.dtype} and {k_weight.dtype}")
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps has to be finite and not below zero, got {eps}")
    return b, s, h, hk, d, table[0]


def _norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions) -> tuple:
    b, s, h, hk, d, rows = _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions)
    dev = _on_one_device(q, k, cos, sin, q_weight, k_weight, positions)
    code = _CODES[q.dtype]
    per = 4 if code == 2 else 8
    q_out, k_out = q.new_empty((b, s, h, d)), k.new_empty((b, s, hk, d))
    cos, sin, q_weight, k_weight = _aligned(cos), _aligned(sin), _aligned(q_weight), _aligned(k_weight)
    if positions is not None:
        positions = positions.contiguous()
    q, *qa = _heads(q, per)
    k, *ka = _heads(k, per)
    _call("tcpxb_norm_rope_forward", dev, _NORM_ROPE.pack(*qa, *ka, _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), _ptr(positions),
                                                          q_out.data_ptr(), k_out.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, b, s, h, hk, d,
                                                          rows, eps, code))
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          eps: float = 1e-6, positions: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dq_weight, dk_weight) of `qk_norm_rope` from the gradients of its outputs and its own
    arguments (the weights' are None without weights).  The same inputs give the same bits every time."""
    b, s, h, hk, d, rows = _check_norm_rope(q, k, cos, sin, q_weight, k_weight, eps, positions)
    for name, t, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if t.shape != x.shape:
            raise ValueError(f"{name} has to be {tuple(x.shape)}, got {tuple(t.shape)}")
        if t.dtype is not x.dtype:
            raise TypeError(f"{name} has to be {x.dtype}, got {t.dtype}")
    dev = _on_one_device(dq_out, dk_out, q, k, cos, sin, q_weight, k_weight, positions)
    code = _CODES[q.dtype]
    per = 4 if code == 2 else 8
    dq, dk = q.new_empty((b, s, h, d)), k.new_empty((b, s, hk, d))
    dwq = dwk = partial = None
    qa = ka = (0, 0, 0, 0)
    if q_weight is not None:
        dwq, dwk = q_weight.new_empty((d,)), k_weight.new_empty((d,))
        partial = cos.new_empty(_entry("tcpxb_norm_rope_scratch_bytes")(d) // 4)
        q, *qa = _heads(q, per)
        k, *ka = _heads(k, per)
    cos, sin, q_weight, k_weight = _aligned(cos), _aligned(sin), _aligned(q_weight), _aligned(k_weight)
    if positions is not None:
        positions = positions.contiguous()
    dq_out, *dqa = _heads(dq_out, per)
    dk_out, *dka = _heads(dk_out, per)
    _call("tcpxb_norm_rope_backward", dev, _NORM_ROPE.pack(*qa, *ka, _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), _ptr(positions), 0, 0,
                                                           *dqa, *dka, dq.data_ptr(), dk.data_ptr(), _ptr(dwq), _ptr(dwk), _ptr(partial), b, s, h, hk, d,
                                                           rows, eps, code))
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
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad) or
                                    (k_weight is not None and k_weight.requires_grad)):
        return _NormRopeFunction.apply(q, k, cos, sin, q_weight, k_weight, eps, positions)
    return _norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions)


# ----------------------------------------------------------------------- AdamW
_data_ptr, _numel, _is_contiguous, _get_device = (getattr(torch.Tensor, n) for n in ("data_ptr", "numel", "is_contiguous", "get_device"))
_dtype = operator.attrgetter("dtype")


def _flat_list(name: str, ts: Sequence[torch.Tensor], numels: Sequence[int], dtype: torch.dtype, device: int) -> list:
    """The tensors' addresses; `device`: -1 stands for the CPU, where the arguments are all that can be checked."""
    if len(ts) != len(numels):
        raise ValueError(f"{len(numels)} tensors, but {len(ts)} {name}")
    if set(map(_dtype, ts)) != {dtype}:
        raise TypeError(f"{name} have to be {dtype}, got {set(map(_dtype, ts))}")
    if list(map(_numel, ts)) != numels:
        i = next(i for i, t in enumerate(ts) if t.numel() != numels[i])
        raise ValueError(f"{name}[{i}] has {ts[i].numel()} elements, not {numels[i]}")
    if not all(map(_is_contiguous, ts)):
        raise ValueError(f"{name} have to be contiguous")
    if set(map(_get_device, ts)) != {device}:
        raise ValueError(f"{name} are on another device")
    return list(map(_data_ptr, ts))


def _table(*columns: Sequence[int]) -> bytes:
    """The C entry's list of tensors: rows of nine words, from lists of each word."""
    return array.array("q", itertools.chain.from_iterable(zip(*columns))).tobytes()


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """Root of the sum of all squares, as a float32 scalar on the device.  Contiguous CUDA tensors of one
    type (bfloat16, float16, float32); squares of a few elements are added in 32 bits, those sums in 64,
    in an order that depends on sizes and alignments alone."""
    grads = list(grads)
    if not grads:
        raise ValueError("no gradients")
    dtype = grads[0].dtype
    if dtype not in _CODES:
        raise TypeError(f"gradients have to be bfloat16, float16 or float32, got {dtype}")
    numels = list(map(_numel, grads))
    at = _flat_list("grads", grads, numels, dtype, grads[0].get_device())
    dev = _on_one_device(grads[0])
    none = [0] * len(grads)
    table = _table(none, at, none, none, none, none, none, none, numels)
    norm = grads[0].new_empty((), dtype=torch.float32)
    scratch = grads[0].new_empty(_entry("tcpxb_grad_norm_scratch_bytes")(table, len(grads)), dtype=torch.uint8)
    _call("tcpxb_grad_norm", dev, table, len(grads), _CODES[dtype], norm.data_ptr(), scratch.data_ptr())
    return norm


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps, *, lr: float, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, max_grad_norm: Optional[float] = None, norm: Optional[torch.Tensor] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
               masters: Optional[Sequence[torch.Tensor]] = None) -> Optional[torch.Tensor]:
    """One AdamW step over all tensors, in place, in two launches (three with clipping).

    `params` and `grads`: contiguous tensors of one type (bfloat16, float16, float32) on one device.
    States in 32 bits: `exp_avgs` and `exp_avg_sqs` are float32 tensors of the params' sizes.  In 8 bits:
    float8_e4m3fn tensors with `exp_avg_scales` and `exp_avg_sq_scales`, one float32 per 256 elements; a
    state's value is code times scale, and `exp_avg_sqs` holds the root.  `steps` (an int32 tensor with an
    entry for each of them, or a list of one-element ones) counts each tensor's updates and is advanced.  `max_grad_norm`: gradients are scaled by
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
    count, device = len(params), params[0].get_device()
    numels = list(map(_numel, params))
    p_at = _flat_list("params", params, numels, dtype, device)
    g_at = _flat_list("grads", grads, numels, dtype, device)
    state = torch.float8_e4m3fn if bits == 8 else torch.float32
    m_at = _flat_list("exp_avgs", exp_avgs, numels, state, device)
    v_at = _flat_list("exp_avg_sqs", exp_avg_sqs, numels, state, device)
    none = [0] * count
    ms_at = vs_at = master_at = none
    written = p_at + m_at + v_at
    if bits == 8:
        blocks = [-(-n // STATE_BLOCK) for n in numels]
        ms_at = _flat_list("exp_avg_scales", list(exp_avg_scales), blocks, torch.float32, device)
        vs_at = _flat_list("exp_avg_sq_scales", list(exp_avg_sq_scales), blocks, torch.float32, device)
        written += ms_at + vs_at
    if masters is not None:
        if dtype is torch.float32:
            raise ValueError("masters stand behind 16-bit params")
        master_at = _flat_list("masters", list(masters), numels, torch.float32, device)
        written += master_at
    if isinstance(steps, torch.Tensor):
        if steps.dtype is not torch.int32:
            raise TypeError(f"steps has to be int32, got {steps.dtype}")
        if steps.shape != (count,) or not steps.is_contiguous() or steps.get_device() != device:
            raise ValueError(f"steps has to be a contiguous [{count}] on the same device, got {tuple(steps.shape)}")
        step_at = steps.data_ptr()
        step_at = range(step_at, step_at + 4 * count, 4)
    else:
        step_at = _flat_list("steps", list(steps), [1] * count, torch.int32, device)
        if len(set(step_at)) != count:
            raise ValueError("a step counter is given twice")
    if 0 in numels:  # a tensor without elements has no address of its own
        written = [x for x, n in zip(written, numels * (len(written) // count)) if n]
    if len(set(written)) != len(written):
        raise ValueError("a tensor is given twice")
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and 0 <= eps < math.inf and 0 <= lr < math.inf and 0 <= weight_decay < math.inf):
        raise ValueError(f"bad numbers: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
    if max_grad_norm is not None and not 0 <= max_grad_norm < math.inf:
        raise ValueError(f"max_grad_norm has to be finite and not below zero, got {max_grad_norm}")
    if norm is not None and (norm.dtype is not torch.float32 or norm.numel() != 1 or max_grad_norm is None):
        raise ValueError("norm has to be one float32 value, given with max_grad_norm")
    dev = _on_one_device(params[0], norm)
    table = _table(p_at, g_at, m_at, v_at, ms_at, vs_at, master_at, step_at, numels)
    compute = max_grad_norm is not None and norm is None
    if compute:
        norm = params[0].new_empty((), dtype=torch.float32)
    scratch = params[0].new_empty(_entry("tcpxb_adamw_scratch_bytes")(table, count), dtype=torch.uint8)
    _call("tcpxb_adamw_step", dev, table, count, _ADAMW.pack(lr, beta1, beta2, eps, weight_decay, _ptr(norm), max_grad_norm or 0.0, compute, bits,
                                                             _CODES[dtype], scratch.data_ptr()))
    if not torch.is_inference_mode_enabled():
        torch.autograd.graph.increment_version(params)  # autograd learns of the update, as of any other in place
    return norm
