"""The training operators in 64 bits, and how far a kernel may be from them.

Tolerances are counted from roundings, element by element.  `half` is half a step of the type, relative
to the value: what one rounding to it can be off.  Roundings to the type are: each operand that a kernel
feeds to the matrix units (probabilities, score gradients) and each result.  Everything else is 32-bit:
a sum of n products is off by at most n 2^-24 of the sum of magnitudes, and the kernels add in pieces,
so n + 8 covers the scaling and the exponential beside it.

Under its normal range a type's steps are all of one size, so an operand is also off by up to half of
its smallest step (`least / 2`), whatever its value: in fp16 that is 2^-25, and a probability of 2^-26
becomes zero.  Such an error enters a product with the other operand's magnitude, summed over the row
(the forward pass's unnormalised probabilities are at least as large as the normalised ones, as their
sum is at least one)."""
import torch

F32 = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def visible(b, sq, sk, causal, lengths):
    ok = torch.ones(b, 1, sq, sk, dtype=torch.bool)
    if causal:
        ok &= torch.arange(sk)[None] <= torch.arange(sq)[:, None] + sk - sq
    if lengths is not None:
        ok &= torch.arange(sk) < lengths.cpu()[:, None, None, None]
    return ok


def attention(q, k, v, dout, causal=False, lengths=None, scale=None):
    """{name: (value, tolerance)} of out, lse, dq, dk and dv, in 64 bits on the CPU or where the inputs are."""
    dtype, (b, sq, h, d), (sk, hk) = q.dtype, q.shape, k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    u = half(dtype)
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    ok = visible(b, sq, sk, causal, lengths).to(q.device)
    at = torch.arange(sk, device=q.device)
    live = (at < lengths.to(q.device)[:, None] if lengths is not None else at.expand(b, sk) >= 0)[:, None, :, None]
    q, dout = (t.double().transpose(1, 2) for t in (q, dout))
    k, v = (torch.where(live, t.double().transpose(1, 2), 0.0).repeat_interleave(h // hk, 1) for t in (k, v))
    s = scale * (q @ k.mT)
    # scores: products, scaling, and the difference to the row's largest in base two
    es = (d + 8) * F32 * scale * (q.abs() @ k.abs().mT)
    s = torch.where(ok, s, -torch.inf)
    top = s.amax(-1, keepdim=True) if sk else s.new_full((b, h, sq, 1), -torch.inf)
    empty = top == -torch.inf
    e = torch.where(ok, (s - torch.where(empty, 0.0, top)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(empty, 1.0, total)
    lse = torch.where(empty, -torch.inf, top + total.clamp_min(1e-300).log()).squeeze(-1)
    # of a probability: its own score's error and the row's, and a few 32-bit steps of exp, sum and division
    rowes = torch.where(ok, es, 0.0).amax(-1, keepdim=True) if sk else torch.zeros_like(top)
    ep = es + rowes + (sk + 16) * F32
    n = max(sq, sk) + 8
    out = p @ v
    mag = p @ v.abs()
    under = (p > 0) * (least / 2)
    eout = u * out.abs() + (u + n * F32) * mag + (p * ep + under) @ v.abs()
    tol = {"out": eout, "lse": rowes.squeeze(-1) + (sk + 16) * F32 + 4 * F32 * lse.abs().nan_to_num(posinf=0.0)}
    dp = dout @ v.mT
    delta = (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edelta = (dout.abs() * eout).sum(-1, keepdim=True) + (d + 8) * F32 * (dout * out).abs().sum(-1, keepdim=True)
    edp = (d + 8) * F32 * (dout.abs() @ v.abs().mT)
    eds = ds.abs() * (u + ep) + p * (1 + u) * (edelta + edp) + under
    dq = scale * (ds @ k)
    edq = u * dq.abs() + scale * ((eds + n * F32 * ds.abs()) @ k.abs())
    dk, dv = scale * (ds.mT @ q), p.mT @ dout
    group = (h // hk) * n * F32
    edk = scale * ((eds + group * ds.abs()).mT @ q.abs())
    edv = (p * (u + ep + group) + under).mT @ dout.abs()

    def shared(x):
        return x.unflatten(1, (hk, h // hk)).sum(2)

    dk, dv = shared(dk), shared(dv)
    vals = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    tol.update(dq=edq, dk=shared(edk) + u * dk.abs(), dv=shared(edv) + u * dv.abs())
    # values under the type's normal range are off by a step of its smallest
    got = {name: (x.transpose(1, 2), tol[name].transpose(1, 2) * 1.001 + least) for name, x in vals.items()}
    got["lse"] = lse, tol["lse"] * 1.001 + 1e-30
    return got


def close(got, want, name):
    """The first element that is further off than it may be, if any."""
    value, tol = want
    got = got.double().to(value.device)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    off = torch.where(same, 0.0, (got - value).abs() - tol)
    bad = ~(off <= 0)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off; at {bad.nonzero()[0].tolist()} {got[bad][0].item()} for {value[bad][0].item()} +- {tol.expand_as(value)[bad][0].item()}"


def rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def norm_rope(x, w, cos, sin, dy, eps, positions=None):
    """{y, dx, dw: (value, tolerance)} for one of queries and keys."""
    dtype, (b, s, h, d) = x.dtype, x.shape
    u = half(dtype)
    at = torch.arange(s, device=x.device).expand(b, s) if positions is None else positions
    cos, sin = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    x, dy = x.double(), dy.double()
    n, r = x, torch.ones_like(x[..., :1])
    if w is not None:
        r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        n = x * r * w.double()
    y = rotate(n, cos, sin)
    # 32-bit: the sum of squares (d products), the root's approximation and four products
    c = (d + 16) * F32
    ey = u * y.abs() + c * rotate(n.abs(), cos.abs(), -sin.abs()).abs() + c * rotate(n.abs(), cos.abs(), sin.abs()).abs()
    dn = rotate(dy, cos, -sin)
    mdn = rotate(dy.abs(), cos.abs(), sin.abs()).abs() + rotate(dy.abs(), cos.abs(), -sin.abs()).abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    if w is None:
        return {"y": (y, ey + tiny), "dx": (dn, u * dn.abs() + c * mdn + tiny)}
    w = w.double()
    xh = x * r
    g = dn * w
    mean = (g * xh).mean(-1, keepdim=True)
    dx = r * (g - xh * mean)
    mag = r * (mdn * w.abs() + xh.abs() * (mdn * w.abs() * xh.abs()).mean(-1, keepdim=True))
    dw = (dn * xh).sum((0, 1, 2))
    edw = u * dw.abs() + (c + (b * s * h + 8) * F32) * (mdn * xh.abs()).sum((0, 1, 2))
    return {"y": (y, ey + tiny), "dx": (dx, u * dx.abs() + 3 * c * mag + tiny), "dw": (dw, edw + tiny)}


E4M3_MAX, BLOCK = 448.0, 256


def adamw(p, g, m, v, step, lr, betas, eps, wd, coef=1.0):
    """(p, m, v) in 64 bits after update number `step`."""
    p, g, m, v = p.double(), g.double() * coef, m.double(), v.double()
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    mh, vh = m / (1 - betas[0] ** step), v / (1 - betas[1] ** step)
    return p * (1 - lr * wd) - lr * mh / (vh.sqrt() + eps), m, v


def dequantise(q, scale):
    return q.double().flatten() * scale.double().repeat_interleave(BLOCK)[:q.numel()]
