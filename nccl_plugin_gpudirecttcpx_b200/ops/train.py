"""Python entry points of the training step's sm_100a operators.

`attention`, `qk_norm_rope` and `adamw_step` (with `grad_norm` and the optimizer `AdamW` on
top) are what a decoder's training step needs next to its gradient collectives.  They take
torch CUDA tensors; a compiled module (`csrc/bind/train_torch.cc`) checks the arguments, makes
outputs and scratch, and passes raw pointers and the device's current stream to the C ABI in
`csrc/include/tcpxb/train.h`.  There is no eager fallback: a missing library is an error.
Arguments are checked on the host before anything is queued: a wrong shape, size or option is
a `ValueError`, a wrong type a `TypeError`.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ..utils import native

STATE_BLOCK = 256  # elements that share a scale of an 8-bit AdamW state

_module = None


def _m():
    global _module
    if _module is None:
        _module = native.module("tcpxb_train_torch")
    return _module


# ------------------------------------------------------------------- attention
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
    Where a wait inside the kernel runs out of time, the rows that it concerns become NaN; with `status`
    (`ops.status_buffer()`) its first word becomes 3, and calls that find a 3 there leave NaN."""
    return _m().attention_forward(q, k, v, causal, scale, key_lengths, status)


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, *,
                       causal: bool = False, scale: Optional[float] = None, key_lengths: Optional[torch.Tensor] = None,
                       status: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dv) from what `attention_forward` returned for the same arguments.  The probabilities
    are computed again from the scores and `lse`.  The same inputs give the same bits every time."""
    return _m().attention_backward(dout, q, k, v, out, lse, causal, scale, key_lengths, status)


class _AttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale, key_lengths):
        out, lse = _m().attention_forward(q, k, v, causal, scale, key_lengths, None)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths)
        ctx.how = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_lengths = ctx.saved_tensors
        causal, scale = ctx.how
        return (*_m().attention_backward(dout, q, k, v, out, lse, causal, scale, key_lengths, None), None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: Optional[float] = None,
              key_lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`attention_forward`'s `out`, differentiable in q, k and v (once)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFunction.apply(q, k, v, causal, scale, key_lengths)
    return _m().attention_forward(q, k, v, causal, scale, key_lengths, None)[0]


# ---------------------------------------------------------------- qk_norm_rope
def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          eps: float = 1e-6, positions: Optional[torch.Tensor] = None) -> tuple:
    """(dq, dk, dq_weight, dk_weight) of `qk_norm_rope` from the gradients of its outputs and its own
    arguments (the weights' are None without weights).  The same inputs give the same bits every time."""
    return _m().norm_rope_backward(dq_out, dk_out, q, k, cos, sin, q_weight, k_weight, eps, positions)


class _NormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, q_weight, k_weight, eps, positions):
        out = _m().norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions)
        normed = q_weight is not None
        # the rotation alone is turned back without its inputs
        ctx.save_for_backward(q if normed else None, k if normed else None, cos, sin, q_weight, k_weight, positions)
        ctx.eps = eps
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, cos, sin, q_weight, k_weight, positions = ctx.saved_tensors
        grads = _m().norm_rope_backward(dq_out, dk_out, dq_out if q is None else q, dk_out if k is None else k, cos, sin, q_weight, k_weight,
                                        ctx.eps, positions)
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
    return _m().norm_rope_forward(q, k, cos, sin, q_weight, k_weight, eps, positions)


# ----------------------------------------------------------------------- AdamW
def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """Root of the sum of all squares, as a float32 scalar on the device.  Contiguous CUDA tensors of one
    type (bfloat16, float16, float32); squares of a few elements are added in 32 bits, those sums in 64,
    in an order that depends on sizes and alignments alone."""
    return _m().grad_norm(list(grads))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps, *, lr: float, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, max_grad_norm: Optional[float] = None, norm: Optional[torch.Tensor] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
               masters: Optional[Sequence[torch.Tensor]] = None) -> Optional[torch.Tensor]:
    """One AdamW step over all tensors, in place.  Up to 380 of them take two launches (three with clipping), longer lists as
    many for each 380.

    `params` and `grads`: contiguous tensors of one type (bfloat16, float16, float32) on one device.
    States in 32 bits: `exp_avgs` and `exp_avg_sqs` are float32 tensors of the params' sizes.  In 8 bits:
    float8_e4m3fn tensors with `exp_avg_scales` and `exp_avg_sq_scales`, one float32 per 256 elements; a
    state's value is code times scale, and `exp_avg_sqs` holds the root.  `steps` (an int32 tensor with an
    entry for each of them, or a list of one-element ones) counts each tensor's updates and is advanced.  `max_grad_norm`: gradients are scaled by
    min(1, max_grad_norm / (norm + 1e-6)), where `norm` is theirs over all tensors (computed here and
    returned), or the given float32 device scalar, for lists that share one.  `masters`: float32 weights
    that are updated and rounded into 16-bit `params`.  Nothing is copied to or from the host: the call can
    be captured into a graph, which then keeps the given numbers and pointers."""
    return _m().adamw_step(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), steps if isinstance(steps, torch.Tensor) else list(steps), lr,
                           *betas, eps, weight_decay, max_grad_norm, norm, None if exp_avg_scales is None else list(exp_avg_scales),
                           None if exp_avg_sq_scales is None else list(exp_avg_sq_scales), None if masters is None else list(masters))
