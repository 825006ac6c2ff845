"""The operators of a training step, as cases whose time can be measured.

A decoder's training step next to the gradient collectives: queries and keys are normalised per head and
rotated, attention runs forward and backward over them, and AdamW updates the weights from the averaged
gradients.  Sizes are those of the data-parallel harness (its full and its toy model, sequences of 2048) and
ranges around them: one token to 8192, head sizes of 16 to 128, padded batches, odd lengths, tensors that are
views of one fused projection, parameter lists from a toy model's to an embedding table's.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 256        # elements that share a scale of an 8-bit state
E4M3_MAX = 448.0
LR, BETA1, BETA2, EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.1
NORM_EPS = 1e-5


def listed():
    return [
        # the toy model of the harness, forward and backward: nothing but latency
        {"name": "attn_train_toy", "op": "attn_train", "dtype": "bf16", "b": 2, "sq": 64, "sk": 64, "h": 4, "hk": 2, "d": 16,
         "causal": True, "padded": False, "fused": False},
        # one layer of the harness's model at its micro-batch, values read out of a fused projection
        {"name": "attn_train_model", "op": "attn_train", "dtype": "bf16", "b": 4, "sq": 2048, "sk": 2048, "h": 32, "hk": 8, "d": 64,
         "causal": True, "padded": False, "fused": True},
        # long sequences with wide heads
        {"name": "attn_train_long", "op": "attn_train", "dtype": "f16", "b": 1, "sq": 8192, "sk": 8192, "h": 16, "hk": 4, "d": 128,
         "causal": True, "padded": False, "fused": False},
        # a padded batch of an encoder: odd length, ragged sequences, every head its own keys
        {"name": "attn_train_padded_odd", "op": "attn_train", "dtype": "bf16", "b": 7, "sq": 777, "sk": 777, "h": 12, "hk": 12, "d": 80,
         "causal": False, "padded": True, "fused": False},
        # evaluation: the forward pass alone, of the same layer
        {"name": "attn_forward_model", "op": "attn_forward", "dtype": "bf16", "b": 4, "sq": 2048, "sk": 2048, "h": 32, "hk": 8, "d": 64,
         "causal": True, "padded": False, "fused": False},
        # the toy model's queries and keys, normalised and rotated, forward and backward
        {"name": "norm_rope_toy", "op": "norm_rope_train", "dtype": "bf16", "b": 2, "s": 64, "h": 4, "hk": 2, "d": 16, "norm": True,
         "fused": False},
        # one layer of the model, forward and backward, out of a fused projection
        {"name": "norm_rope_train_model", "op": "norm_rope_train", "dtype": "bf16", "b": 4, "s": 2048, "h": 32, "hk": 8, "d": 64,
         "norm": True, "fused": True},
        # the rotation alone (the model has no head norms by default), 32-bit values, an odd length, forward
        {"name": "rope_forward_odd_f32", "op": "norm_rope_forward", "dtype": "f32", "b": 3, "s": 1777, "h": 16, "hk": 4, "d": 128,
         "norm": False, "fused": False},
        # the toy model's whole parameter list with clipping: launches and Python
        {"name": "adamw_toy_clip", "op": "adamw", "dtype": "bf16", "layers": 2, "dim": 64, "kv": 32, "ffn": 128, "vocab": 512, "odd": 0,
         "bits": 32, "clip": True},
        # embedding table and one layer of the model, states in 32 bits, gradients clipped by their global norm
        {"name": "adamw_model_clip", "op": "adamw", "dtype": "bf16", "layers": 1, "dim": 2048, "kv": 512, "ffn": 8192, "vocab": 128256,
         "odd": 0, "bits": 32, "clip": True},
        # the same with states in 8 bits
        {"name": "adamw_model_8bit", "op": "adamw", "dtype": "bf16", "layers": 1, "dim": 2048, "kv": 512, "ffn": 8192, "vocab": 128256,
         "odd": 0, "bits": 8, "clip": False},
        # 32-bit weights whose sizes leave every following gradient of the bucket off the vector boundary
        {"name": "adamw_odd_f32", "op": "adamw", "dtype": "f32", "layers": 2, "dim": 1000, "kv": 250, "ffn": 2001, "vocab": 3001, "odd": 1,
         "bits": 32, "clip": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("attn_train", "attn_train", "attn_forward", "norm_rope_train", "norm_rope_forward", "adamw"))
    if op == "adamw":
        dim = _log(rng, 32, 2048)
        return {"op": op, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "layers": 1, "dim": dim, "kv": max(1, dim // rng.choice((1, 2, 4, 8))),
                "ffn": _log(rng, dim, 4 * dim), "vocab": _log(rng, 256, 65536), "odd": rng.choice((0, 0, 1, 3)),
                "bits": rng.choice((32, 8)), "clip": rng.random() < 0.5}
    hk, group = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 3, 4, 8))
    d = 8 * rng.randint(2, 16) if rng.random() < 0.4 else rng.choice((64, 128))
    dtype = rng.choice(("bf16", "bf16", "f16") if op.startswith("attn") else ("bf16", "f16", "f32"))
    s, b = _log(rng, 1, 8192), _log(rng, 1, 16)
    if op.startswith("norm"):
        h = hk * max(1, min(group, (1 << 24) // (s * hk * d)))
        return {"op": op, "dtype": dtype, "b": max(1, min(b, (1 << 24) // (s * h * d))), "s": s, "h": h, "hk": hk, "d": d,
                "norm": rng.random() < 0.7, "fused": rng.random() < 0.5}
    # with a single key the scores have no gradient: what two sides leave there is rounding and cannot be compared
    least = 2 if op == "attn_train" else 1
    s = max(s, least)
    sk = s if rng.random() < 0.7 else _log(rng, least, 8192)
    h = hk * max(1, min(group, (1 << 29) // (s * sk * hk)))
    return {"op": op, "dtype": dtype, "b": max(1, min(b, (1 << 29) // (s * sk * h))), "sq": s, "sk": sk, "h": h, "hk": hk, "d": d,
            "causal": rng.random() < 0.6, "padded": rng.random() < 0.4, "fused": sk == s and rng.random() < 0.4}


def _shapes(c):
    """The parameter list of a decoder with `layers` layers; `odd` makes every size a little larger."""
    o, dim = c["odd"], c["dim"]
    layer = [(dim + o,), (dim + o,), (dim, dim + o), (c["kv"], dim + o), (c["kv"], dim + o), (dim, dim + o),
             (c["ffn"], dim + o), (c["ffn"], dim + o), (dim, c["ffn"] + o)]
    return [(c["vocab"], dim + o)] + layer * c["layers"] + [(dim + o,)]


def _blocks(flat):
    n = -flat.numel() % BLOCK
    return torch.nn.functional.pad(flat, (0, n)).view(-1, BLOCK)


def _quantise(x, root):
    """Values in e4m3 and a 32-bit scale per block.  Of a root, what is above zero stays above zero."""
    b = _blocks(x.reshape(-1))
    top = b.abs().amax(1, keepdim=True)
    held = top >= 1e-30
    t = b * torch.where(held, E4M3_MAX / top, torch.zeros_like(top))
    if root:
        t = torch.where(t > 0, t.clamp_min(2.0 ** -9), t)
    scale = torch.where(held, top / E4M3_MAX, torch.zeros_like(top)).view(-1)
    return t.view(-1)[:x.numel()].to(torch.float8_e4m3fn).view(x.shape), scale


def _dequantise(q, scale):
    return (_blocks(q.reshape(-1).to(scale.dtype)) * scale[:, None]).view(-1)[:q.numel()].view(q.shape)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g).to(dt)

    s = dict(case)
    if op == "adamw":
        shapes = _shapes(case)
        counts = [math.prod(x) for x in shapes]

        def flat(std):
            # weights and gradients of a list lie one behind another, as in a bucket of the harness
            values = torch.randn(sum(counts), device=dev, generator=g).mul_(std).to(dt)
            return [t.view(x) for t, x in zip(values.split(counts), shapes)]

        s["params"], s["grads"] = flat(0.02), flat(1e-3)
        m = [torch.randn(x, device=dev, generator=g).mul_(3e-4) for x in shapes]
        v = [torch.randn(x, device=dev, generator=g).mul_(1e-3).square_() for x in shapes]
        s["steps"] = torch.full((len(shapes),), 100, dtype=torch.int32, device=dev)
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
        else:
            s["m"], s["m_scale"] = zip(*[_quantise(x, False) for x in m])
            s["v"], s["v_scale"] = zip(*[_quantise(x.sqrt(), True) for x in v])
        return s
    b, h, hk, d = case["b"], case["h"], case["hk"], case["d"]
    sq, sk = case.get("sq", case.get("s")), case.get("sk", case.get("s"))
    if case["fused"]:
        s["q"], s["k"], s["v"] = normal(b, sq, h + 2 * hk, d).split((h, hk, hk), 2)
    else:
        s["q"], s["k"], s["v"] = normal(b, sq, h, d), normal(b, sk, hk, d), normal(b, sk, hk, d)
    if op.startswith("norm"):
        inv = 500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = torch.arange(sq, device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["wq"], s["wk"] = ((1 + 0.1 * normal(d)).to(dt), (1 + 0.1 * normal(d)).to(dt)) if case["norm"] else (None, None)
        s["dq"], s["dk"] = normal(b, sq, h, d), normal(b, sq, hk, d)
        return s
    s["dout"] = normal(b, sq, h, d)
    # lengths of a padded batch: the longest sequence fills it
    lens = torch.randint(0, sk + 1, (b,), device=dev, generator=g, dtype=torch.int32)
    lens[0] = sk
    s["lens"] = lens if case["padded"] else None
    return s


def _valid(s, sq, sk, dev):
    """[batch or 1, 1, 1, sq, sk]: which keys a query sees."""
    j = torch.arange(sk, device=dev)
    ok = torch.ones(1, 1, 1, sq, sk, dtype=torch.bool, device=dev)
    if s["causal"]:
        ok = ok & (j <= torch.arange(sq, device=dev)[:, None] + (sk - sq))
    if s["lens"] is not None:
        ok = ok & (j < s["lens"][:, None, None, None, None])
    return ok


def _attention(s, train):
    q, k, v = s["q"], s["k"], s["v"]
    (b, sq, h, d), (_, sk, hk, _) = q.shape, k.shape
    scale = d ** -0.5
    q5 = q.float().view(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    k5, v5 = (x.float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    p = q5 @ k5.transpose(-1, -2)
    p.mul_(scale).masked_fill_(~_valid(s, sq, sk, q.device), -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = p @ v5

    def back(x):
        return x.permute(0, 3, 1, 2, 4).reshape(b, sq, h, d).to(q.dtype)

    if not train:
        return back(o)
    do = s["dout"].float().view(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = do @ v5.transpose(-1, -2)
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq = ds @ k5
    dk = (ds.transpose(-1, -2) @ q5).sum(2)
    return back(o), back(dq), dk.permute(0, 2, 1, 3).to(q.dtype).contiguous(), dv.permute(0, 2, 1, 3).to(q.dtype).contiguous()


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _norm_rope(x, w, cos, sin):
    n = x.float()
    if w is not None:
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + NORM_EPS) * w.float()
    return _rotate(n, cos, sin).to(x.dtype)


def _norm_rope_backward(dy, x, w, cos, sin):
    dn = _rotate(dy.float(), cos, -sin)
    if w is None:
        return dn.to(x.dtype), None
    f = x.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + NORM_EPS)
    xh = f * r
    dxh = dn * w.float()
    dx = r * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))
    dw = (dn * xh).sum((0, 1, 2), dtype=torch.float64)
    return dx.to(x.dtype), dw.to(w.dtype)


def _adamw(s):
    g32 = [g.float() for g in s["grads"]]
    if s["clip"]:
        norm = torch.stack([g.square().sum(dtype=torch.float64) for g in g32]).sum().sqrt().float()
        coef = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
        g32 = [g * coef for g in g32]
    s["steps"] += 1
    t = s["steps"].double()
    c1, c2 = (1 - BETA1 ** t).unbind(), (1 - BETA2 ** t).unbind()
    if s["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = [_dequantise(q, c) for q, c in zip(s["m"], s["m_scale"])]
        v = [_dequantise(q, c).square() for q, c in zip(s["v"], s["v_scale"])]
    m = [x.mul(BETA1) + (1 - BETA1) * g for x, g in zip(m, g32)]
    v = [x.mul(BETA2) + (1 - BETA2) * g * g for x, g in zip(v, g32)]
    new = [p.float() * (1 - LR * DECAY) - (LR / a).float() * x / (y.sqrt() / b.sqrt().float() + EPS)
           for p, x, y, a, b in zip(s["params"], m, v, c1, c2)]
    [p.copy_(x) for p, x in zip(s["params"], new)]
    if s["bits"] == 32:
        [a.copy_(x) for a, x in zip(s["m"], m)]
        [a.copy_(x) for a, x in zip(s["v"], v)]
        return _outputs(s)
    [(a.copy_(x), c.copy_(y)) for a, c, (x, y) in zip(s["m"], s["m_scale"], [_quantise(x, False) for x in m])]
    [(a.copy_(x), c.copy_(y)) for a, c, (x, y) in zip(s["v"], s["v_scale"], [_quantise(x.sqrt(), True) for x in v])]
    return _outputs(s)


def _outputs(s):
    out = {"params": list(s["params"]), "m": list(s["m"]), "v": list(s["v"])}
    if s["bits"] == 8:
        # the values in units of their blocks' scales, and the scales
        out.update(m_scale=list(s["m_scale"]), v_scale=list(s["v_scale"]))
    return out


def run(s):
    op = s["op"]
    if own:
        from nccl_plugin_gpudirecttcpx_b200 import ops
        if op == "adamw":
            ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["steps"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                           weight_decay=DECAY, max_grad_norm=1.0 if s["clip"] else None, exp_avg_scales=s.get("m_scale"),
                           exp_avg_sq_scales=s.get("v_scale"))
            return _outputs(s)
        if op.startswith("norm"):
            args = s["cos"], s["sin"], s["wq"], s["wk"]
            q, k = ops.qk_norm_rope(s["q"], s["k"], *args, eps=NORM_EPS)
            if op == "norm_rope_forward":
                return q, k
            return q, k, ops.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], *args, eps=NORM_EPS)
        how = {"causal": s["causal"], "key_lengths": s["lens"]}
        if op == "attn_forward":
            return ops.attention(s["q"], s["k"], s["v"], **how)
        out, lse = ops.attention_forward(s["q"], s["k"], s["v"], **how)
        return (out, *ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how))
    if op == "adamw":
        return _adamw(s)
    if op.startswith("norm"):
        cos, sin = s["cos"][:, None], s["sin"][:, None]
        q, k = _norm_rope(s["q"], s["wq"], cos, sin), _norm_rope(s["k"], s["wk"], cos, sin)
        if op == "norm_rope_forward":
            return q, k
        (dq, dwq), (dk, dwk) = (_norm_rope_backward(s["dq"], s["q"], s["wq"], cos, sin),
                                _norm_rope_backward(s["dk"], s["k"], s["wk"], cos, sin))
        return q, k, (dq, dk, dwq, dwk)
    return _attention(s, op == "attn_train")


def work(case):
    """Inputs read once, outputs written once; four operations per head element and visible pair forward, ten backward
    (the recomputed scores are the kernel's own affair: the forward pass's are counted once)."""
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "adamw":
        n = sum(math.prod(x) for x in _shapes(case))
        state = 4 * 4 if case["bits"] == 32 else 4 * (1 + 4 / BLOCK)
        return {"bytes": n * (3 * size + state), "flops": 14 * n}
    b, h, hk, d = case["b"], case["h"], case["hk"], case["d"]
    if case["op"].startswith("norm"):
        n = b * case["s"] * (h + hk) * d
        train = case["op"] == "norm_rope_train"
        # forward x -> y; backward x, dy -> dx, where x is read once
        return {"bytes": n * size * (4 if train else 2) + case["s"] * d * 4, "flops": n * (8 + 14 * train)}
    sq, sk = case["sq"], case["sk"]
    # a padded batch's lengths are uniform between nothing and everything, the first sequence whole
    share = (1 + (b - 1) / 2) / b if case["padded"] else 1.0
    if case["causal"]:
        first = sk - sq + 1  # keys that the first query sees, where above zero
        pairs = sq * (first + sk) / 2 if first > 0 else sk * (sk + 1) / 2
    else:
        pairs = sq * sk
    flops = 4 * d * b * h * pairs * share
    q, kv = b * sq * h * d, b * sk * hk * d * share
    if case["op"] == "attn_forward":
        return {"bytes": size * (2 * q + 2 * kv), "flops": flops}
    return {"bytes": size * (4 * q + 4 * kv), "flops": 3.5 * flops}


def _exact_attention(s, train):
    """Head by head through autograd of the definition in 64 bits."""
    (b, sq, h, d), hk = s["q"].shape, s["k"].shape[2]
    outs = [torch.zeros(s[n].shape, dtype=torch.float64, device=s["q"].device) for n in ("q", "q", "k", "v")]
    sk = s["k"].shape[1]
    rows, cols = torch.arange(sq, device=s["q"].device), torch.arange(sk, device=s["q"].device)
    for i in range(b):
        seen = torch.ones(sq, sk, dtype=torch.bool, device=rows.device)
        if s["causal"]:
            seen &= rows[:, None] + (sk - sq) >= cols[None]
        if s["lens"] is not None:
            seen &= (cols < s["lens"][i])[None]
        bias = torch.where(seen, 0.0, -torch.inf).double()
        alive = seen.any(1)
        for j in range(h):
            kv = j // (h // hk)
            x = [s["q"][i, :, j], s["k"][i, :, kv], s["v"][i, :, kv]]
            x = [t.double().requires_grad_(train) for t in x]
            # rows that see nothing take a uniform softmax that is then thrown away
            z = x[0] @ x[1].T / math.sqrt(d) + torch.where(alive[:, None], bias, torch.zeros_like(bias))
            o = torch.softmax(z, 1) @ x[2] * alive[:, None]
            outs[0][i, :, j] = o.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(o, x, s["dout"][i, :, j].double())
                outs[1][i, :, j] = dq
                outs[2][i, :, kv] += dk
                outs[3][i, :, kv] += dv
    return tuple(outs) if train else outs[0]


def _exact_norm_rope(s, train):
    turn = torch.complex(s["cos"].double(), s["sin"].double())[None, :, None]

    def y(x, w):
        n = x if w is None else x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + NORM_EPS).sqrt() * w
        return torch.view_as_real(torch.view_as_complex(n.reshape(*n.shape[:-1], -1, 2)) * turn).flatten(-2)

    got, grads = [], []
    for x, w, dy in ((s["q"], s["wq"], s["dq"]), (s["k"], s["wk"], s["dk"])):
        leaves = [t.double().requires_grad_() for t in (x, w) if t is not None]
        out = y(leaves[0], leaves[1] if w is not None else None)
        got.append(out.detach())
        grads.append(torch.autograd.grad(out, leaves, dy.double()) if train else None)
    if not train:
        return tuple(got)
    (dq, *dwq), (dk, *dwk) = grads
    return got[0], got[1], (dq, dk, dwq[0] if dwq else None, dwk[0] if dwk else None)


def _exact_adamw(s):
    clip = 1.0
    if s["clip"]:
        clip = min(1.0, 1.0 / (math.sqrt(sum(float(g.double().pow(2).sum()) for g in s["grads"])) + 1e-6))
    out = {"params": [], "m": [], "v": [], "m_scale": [], "v_scale": []}
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        t = int(s["steps"][i]) + 1
        p, g = p.double(), g.double() * clip
        if s["bits"] == 32:
            m, v = s["m"][i].double(), s["v"][i].double()
        else:
            m = _dequantise(s["m"][i], s["m_scale"][i].double())
            v = _dequantise(s["v"][i], s["v_scale"][i].double()).pow(2)
        m = m + (g - m) * (1 - BETA1)
        v = v + (g.pow(2) - v) * (1 - BETA2)
        step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["params"].append(p - LR * (DECAY * p + step))
        if s["bits"] == 32:
            out["m"].append(m)
            out["v"].append(v)
            continue
        for x, name in ((m, "m"), (v.sqrt(), "v")):
            x = x.flatten()
            parts = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).reshape(-1, BLOCK)
            scale = parts.abs().max(1).values / E4M3_MAX
            # what the state holds is known only as codes: no value in 64 bits, the scales have one
            out[name].append(None)
            out[name + "_scale"].append(scale)
    return out if s["bits"] == 8 else {n: out[n] for n in ("params", "m", "v")}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"].startswith("norm"):
        return _exact_norm_rope(s, case["op"] == "norm_rope_train")
    if case["b"] * case["h"] > 1024:
        return None  # a loop over heads would take too long
    return _exact_attention(s, case["op"] == "attn_train")
