"""AdamW over many tensors and the gradients' norm against the formulas in 64 bits."""
import math

import pytest
import torch

import train_oracle as oracle
from nccl_plugin_gpudirecttcpx_b200 import ops

gpu = pytest.mark.gpu
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HOW = {"lr": 1e-2, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}
SIZES = [1, 0, 255, 256, 257, 8191, 8192, 8193, 3 * 8192 + 7, 40000, 5]


def tensors(sizes, dtype, bits=32, master=False, seed=0, offset=0, steps=6, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)

    def flat(std, dt):
        # views of one buffer, `offset` elements into it: every alignment there is
        buf = torch.randn(sum(sizes) + offset, device=device, generator=g).mul_(std).to(dt)
        return list(buf[offset:].split(sizes))

    s = {"params": flat(0.5, dtype), "grads": flat(0.1, dtype), "steps": torch.full((len(sizes),), steps, dtype=torch.int32, device=device)}
    m, v = flat(0.05, F32), [x.square() for x in flat(0.1, F32)]
    if bits == 32:
        s["exp_avgs"], s["exp_avg_sqs"] = m, v
    else:
        for name, xs in (("exp_avg", m), ("exp_avg_sq", [x.sqrt() for x in v])):
            pads = [torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256) for x in xs]
            s[name + "_scales"] = [x.abs().amax(1) / 448 for x in pads]
            s[name + "s"] = [(x / c.clamp_min(1e-30)[:, None]).flatten()[:n].to(E4M3) for x, c, n in zip(pads, s[name + "_scales"], sizes)]
    if master:
        s["masters"] = [p.float() + 1e-4 * torch.randn(p.shape, device=device, generator=g) for p in s["params"]]
    return s


def state(s, i):
    if "exp_avg_scales" not in s:
        return s["exp_avgs"][i].double(), s["exp_avg_sqs"][i].double()
    return (oracle.dequantise(s["exp_avgs"][i], s["exp_avg_scales"][i]), oracle.dequantise(s["exp_avg_sqs"][i], s["exp_avg_sq_scales"][i]).square())


def step_and_check(s, how=HOW, max_grad_norm=None):
    before = {n: [t.clone() for t in ts] for n, ts in s.items()}
    old = [state(before, i) for i in range(len(s["params"]))]
    norm = ops.adamw_step(**s, **how, max_grad_norm=max_grad_norm)
    coef = 1.0
    if max_grad_norm is not None:
        exact = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
        # 32 squares of a thread, added in 32 bits; the rest in 64
        assert abs(norm.item() - exact) <= 40 * oracle.F32 * exact + 1e-44
        coef = min(1.0, max_grad_norm / (norm.item() + 1e-6))
    dtype = s["params"][0].dtype
    for i, (p, g) in enumerate(zip(before["params"], before["grads"])):
        assert s["steps"][i] == before["steps"][i] + 1 and torch.equal(s["grads"][i], g)
        start = before["masters"][i] if "masters" in s else p
        b1, b2 = how["betas"]
        want_p, want_m, want_v = oracle.adamw(start, g, *old[i], int(s["steps"][i]), coef=coef, **{n: how[n] for n in ("lr", "betas", "eps")}, wd=how["weight_decay"])
        # m and v: the numbers' own rounding (1 - b in 32 bits is off by up to 2^-24 absolute), the products and the sum
        em = 6 * oracle.F32 * ((b1 * old[i][0]).abs() + g.double().abs() * coef) + 1e-44
        ev = 6 * oracle.F32 * (old[i][1] + (g.double() * coef).square()) + 1e-44
        move = (want_p - start.double() * (1 - how["lr"] * how["weight_decay"])).abs()
        root = (want_v / (1 - b2 ** int(s["steps"][i]))).sqrt() + how["eps"]
        corr = how["lr"] / (1 - b1 ** int(s["steps"][i]))
        rel_root = 0.5 * ev / want_v.clamp_min(1e-40) + 8 * oracle.F32
        ep = 4 * oracle.F32 * start.double().abs() + move * (rel_root + 8 * oracle.F32) + corr * em / root + 1e-44
        if "masters" in s:
            oracle.close(s["masters"][i], (want_p, ep), "master")
            assert torch.equal(s["params"][i], s["masters"][i].to(dtype))
        else:
            tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            oracle.close(s["params"][i], (want_p, ep * (1 + 1e-3) + oracle.half(dtype) * (want_p.abs() + ep) * (dtype != F32) + tiny), "param")
        if "exp_avg_scales" not in s:
            oracle.close(s["exp_avgs"][i], (want_m, em), "exp_avg")
            oracle.close(s["exp_avg_sqs"][i], (want_v, ev), "exp_avg_sq")
            continue
        for codes, scales, want in ((s["exp_avgs"][i], s["exp_avg_scales"][i], want_m), (s["exp_avg_sqs"][i], s["exp_avg_sq_scales"][i], want_v.sqrt())):
            if not want.numel():
                continue
            blocks = torch.nn.functional.pad(want, (0, -want.numel() % 256)).view(-1, 256)
            top = blocks.abs().amax(1) / 448
            oracle.close(scales, (top, top * 2.0 ** -18 + (em if want is want_m else 0 * em).max() / 448), "scale")
            unit = top.repeat_interleave(256)[:want.numel()]
            # half a step of the code, which is 2^-4 of the value and never under half the smallest code (2^-10 units);
            # a root above zero may be raised to that smallest code
            off = want.abs() * 2.0 ** -4 + unit * (2.0 ** -10 if want is want_m else 2.0 ** -9)
            oracle.close(oracle.dequantise(codes, scales), (want, off * (1 + 1e-4) + 1e-40), "code")
    return norm


@gpu
@pytest.mark.parametrize("dtype,master", [(BF16, False), (F16, False), (F32, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_against_the_formula(dtype, master, bits, offset):
    s = tensors(SIZES, dtype, bits, master, seed=offset, offset=offset)
    for _ in range(2):
        step_and_check(s)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("limit", [0.5, 1e6])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_clipping(dtype, bits, limit):
    step_and_check(tensors(SIZES, dtype, bits, seed=1), max_grad_norm=limit)


@gpu
@pytest.mark.parametrize("count", [1, 24, 25, 380, 381, 1000])
def test_long_lists(count):
    """More tensors than one launch's parameters hold; shared and given norms."""
    sizes = [(i * 37) % 700 for i in range(count)]
    norm = step_and_check(tensors(sizes, F32, seed=2), max_grad_norm=0.1)
    s = tensors(sizes, F32, seed=2)
    assert torch.equal(ops.grad_norm(s["grads"]), norm)
    given = ops.adamw_step(**s, **HOW, max_grad_norm=0.1, norm=norm)
    assert given is norm


@gpu
def test_first_steps_and_single_values():
    s = tensors([1, 300], F32, seed=3, steps=0)
    for x in s["exp_avgs"] + s["exp_avg_sqs"]:
        x.zero_()
    for _ in range(3):
        step_and_check(s)
    step_and_check(tensors([300], F32, seed=4, steps=0), {**HOW, "betas": (0.0, 0.0)})
    step_and_check(tensors([300], F32, seed=4, steps=1 << 20), {**HOW, "weight_decay": 0.0, "lr": 0.0})


@gpu
def test_autograd_learns_of_the_update():
    s = tensors([300], F32, seed=10)
    w = s["params"][0].requires_grad_()
    loss = (w * w).sum()
    with torch.no_grad():
        ops.adamw_step(**s, **HOW)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_keep_everything_finite(bits):
    s = tensors([1000], BF16, bits, seed=5, steps=0)
    for n, ts in s.items():
        if n not in ("params", "steps"):
            for t in ts:
                t.view(torch.uint8).zero_()
    step_and_check(s)
    assert all(t.float().isfinite().all() for n in ("params", "exp_avgs", "exp_avg_sqs") for t in s[n])
    assert not s["exp_avgs"][0].float().any()


@gpu
def test_small_roots_stay_above_zero_in_8_bits():
    """One large and many small second moments in a block: no element is left with a root of zero."""
    s = tensors([256], F32, 8, seed=6, steps=0)
    for n in ("exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"):
        s[n][0].view(torch.uint8).zero_()
    s["grads"][0].fill_(1e-8)
    s["grads"][0][7] = 1.0
    before = s["params"][0].clone()
    for _ in range(3):
        ops.adamw_step(**s, **{**HOW, "lr": 1e-3})
    assert (s["exp_avg_sqs"][0].float() > 0).all()
    assert ((s["params"][0] - before).abs() < 0.02).all()


@gpu
@pytest.mark.parametrize("dtype,master", [(BF16, False), (F16, False), (F32, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset,eps", [(0, 0.0), (1, 0.0), (0, 1e-15), (8, 1e35)])
def test_eps_of_the_kernels_with_quotients(dtype, master, bits, offset, eps):
    s = tensors(SIZES, dtype, bits, master, seed=30 + offset, offset=offset)
    for _ in range(2):
        step_and_check(s, {**HOW, "eps": eps})
    many = tensors([300] * 30, dtype, bits, master, seed=31)
    step_and_check(many, {**HOW, "eps": eps}, max_grad_norm=0.5)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-39, 1e-30, 1e-20, 1e-18, 1e-12, 1e-10, 1e33])
def test_small_second_moments_and_extreme_eps(bits, eps):
    """Second moments under the 32-bit normal range (1e-39 to 1e-35 here) are the denominator's own part where `eps` is
    none: a first step is then about the learning rate, as the formula has it."""
    s = tensors([700], F32, bits, seed=18, steps=0)
    for n in ("exp_avgs", "exp_avg_sqs") + (("exp_avg_scales", "exp_avg_sq_scales") if bits == 8 else ()):
        s[n][0].view(torch.uint8).zero_()
    sign = s["grads"][0].sign()
    s["grads"][0].copy_(sign * torch.logspace(-18, -16, 700, device="cuda"))
    how = {**HOW, "betas": (0.9, 0.999), "eps": eps}
    before = s["params"][0].clone()
    step_and_check(s, how)
    if eps <= 1e-30:
        # lr times |g| / |g|, off by the moments' few roundings (a v of 1e-39 has steps of 1.4e-45); the rest is the decay
        assert ((before * (1 - 1e-3) - s["params"][0]) / sign - 1e-2).abs().max() < 1e-6
    if 0 < eps < 1:
        # nothing has moved yet, nothing moves: zero over a denominator whose reciprocal is out of range is zero
        for t in s["grads"] + s["exp_avgs"] + s["exp_avg_sqs"] + s.get("exp_avg_scales", []) + s.get("exp_avg_sq_scales", []):
            t.view(torch.uint8).zero_()
        step_and_check(s, how)
        assert s["params"][0].isfinite().all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_bad_gradients_show(bits, bad):
    """They reach their own element (in 8 bits an infinity its block), and with clipping everything."""
    s = tensors([1024, 512], F32, bits, seed=7)
    s["grads"][0][300] = bad
    clip = tensors([1024, 512], F32, bits, seed=7)
    clip["grads"][0][300] = bad
    ops.adamw_step(**s, **HOW)
    assert s["params"][0][300].isnan() and s["params"][0].isnan().sum() == 1 and s["params"][1].isfinite().all()
    assert state(s, 0)[0][:256].isfinite().all() and state(s, 0)[0][512:].isfinite().all() and not state(s, 0)[0][300].isfinite()
    norm = ops.adamw_step(**clip, **HOW, max_grad_norm=1.0)
    assert not norm.isfinite()


@gpu
def test_norm():
    for dtype in (BF16, F16, F32):
        for sizes in ([0], [1], SIZES, [1 << 22]):
            g = tensors(sizes, dtype, seed=8, offset=1)["grads"]
            exact = math.sqrt(sum(float(x.double().square().sum()) for x in g))
            assert abs(ops.grad_norm(g).item() - exact) <= 40 * oracle.F32 * exact
    g = [torch.full((100,), 3e18, device="cuda"), torch.full((100,), 1e-30, device="cuda")]
    assert abs(ops.grad_norm(g).item() - 3e19) <= 1e-5 * 3e19


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_every_time_and_in_a_graph(bits):
    """A captured step advances its counters with every replay and gives what eager steps give."""
    eager, again, graph = (tensors(SIZES, BF16, bits, seed=9) for _ in range(3))
    for _ in range(3):
        ops.adamw_step(**eager, **HOW, max_grad_norm=0.3)
        ops.adamw_step(**again, **HOW, max_grad_norm=0.3)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.adamw_step(**graph, **HOW, max_grad_norm=0.3)
    for _ in range(3):
        g.replay()
    for n in eager:
        for a, b, c in zip(eager[n], again[n], graph[n]):
            assert torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)
            assert torch.equal(a.view(torch.uint8) if a.dim() else a, c.view(torch.uint8) if c.dim() else c)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_several_lists_one_after_another(bits):
    """Kernels that are set up while the one before them ends: gradients written right before a step, steps and norms
    behind one another without a pause, eager and in a graph, against the same with a pause after every call."""
    sizes = [(i * 61) % 900 for i in range(800)] + [300000]
    paused, eager, graph = (tensors(sizes, BF16, bits, seed=14) for _ in range(3))
    sources = [tensors(sizes, BF16, bits, seed=s)["grads"] for s in (15, 16, 17)]

    def run(s, pause):
        norms = []
        for grads in sources:
            torch._foreach_copy_(s["grads"], grads)
            pause()
            norms.append(ops.adamw_step(**s, **HOW, max_grad_norm=0.3))
            pause()
            norms.append(ops.grad_norm(s["grads"]))
            pause()
        return norms

    wanted = run(paused, torch.cuda.synchronize)
    norms = [run(eager, lambda: None)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norms.append(run(graph, lambda: None))
    g.replay()
    for other, found in zip((eager, graph), norms):
        assert all(torch.equal(a, b) for a, b in zip(wanted, found))
        for n in paused:
            assert all(torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8)) for a, b in zip(paused[n], other[n]))


def test_refusals():
    def call(change=(), **kw):
        s = tensors([10, 300], BF16, device="cpu")
        s.update(change)
        ops.adamw_step(**s, **{**HOW, **kw})

    s = tensors([10, 300], BF16, device="cpu")
    s8 = tensors([10, 300], BF16, 8, device="cpu")
    wide = [torch.zeros(10, dtype=BF16), torch.zeros(300, 2, dtype=BF16)[:, 0]]
    for kind, change, kw in [
        (ValueError, {"params": []}, {}),
        (TypeError, {"params": [p.double() for p in s["params"]]}, {}),
        (TypeError, {"grads": [g.float() for g in s["grads"]]}, {}),
        (ValueError, {"grads": s["grads"][:1]}, {}),
        (ValueError, {"grads": s["grads"][::-1]}, {}),
        (ValueError, {"grads": wide}, {}),
        (ValueError, {"params": wide}, {}),
        (TypeError, {"exp_avgs": [m.bfloat16() for m in s["exp_avgs"]]}, {}),
        (ValueError, {"exp_avg_scales": s8["exp_avg_scales"]}, {}),
        (TypeError, {"exp_avg_scales": s8["exp_avg_scales"], "exp_avg_sq_scales": s8["exp_avg_sq_scales"]}, {}),
        (ValueError, {**s8, "exp_avg_scales": s8["exp_avg_scales"][::-1]}, {}),
        (ValueError, {"masters": s["exp_avgs"][:1]}, {}),
        (TypeError, {"masters": s["params"]}, {}),
        (TypeError, {"steps": s["steps"].long()}, {}),
        (ValueError, {"steps": s["steps"][:1]}, {}),
        (ValueError, {"exp_avgs": s["exp_avg_sqs"], "exp_avg_sqs": s["exp_avg_sqs"]}, {}),
        (ValueError, {}, {"lr": -1.0}),
        (ValueError, {}, {"lr": math.nan}),
        (ValueError, {}, {"betas": (1.0, 0.9)}),
        (ValueError, {}, {"eps": -1.0}),
        (ValueError, {}, {"weight_decay": math.inf}),
        (ValueError, {}, {"max_grad_norm": -1.0}),
        (ValueError, {}, {"norm": torch.zeros(())}),
        (ValueError, {}, {"norm": torch.zeros(2), "max_grad_norm": 1.0}),
        (ValueError, {}, {}),  # not on a GPU
    ]:
        with pytest.raises(kind):
            call(change, **kw)
    with pytest.raises(ValueError):
        twice = tensors([300, 300], F32, device="cpu")
        twice["params"][1] = twice["params"][0]
        ops.adamw_step(**twice, **HOW)
    with pytest.raises(ValueError):
        tensors32 = tensors([300], F32, device="cpu")
        ops.adamw_step(**tensors32, **HOW, masters=tensors32["exp_avgs"])
    for kind, grads in ((ValueError, []), (TypeError, [torch.zeros(3, dtype=torch.float64)]), (TypeError, [torch.zeros(3), torch.zeros(3, dtype=BF16)]),
                        (ValueError, [torch.zeros(3)])):
        with pytest.raises(kind):
            ops.grad_norm(grads)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_share_memory_are_refused(bits):
    """Views that overlap by an element, at their beginning, end or inside; a gradient, counter or norm that is also written."""
    def refused(match="shares memory", **change):
        s = tensors([300, 300], F32, bits, device="cpu")
        s.update(change)
        with pytest.raises(ValueError, match=match):
            ops.adamw_step(**s, **{**HOW, **({"max_grad_norm": 1.0} if "norm" in change else {})})

    buf = torch.zeros(1000)
    codes = buf.to(tensors([1], F32, bits, device="cpu")["exp_avgs"][0].dtype)
    for a, b in ((0, 299), (299, 0), (5, 5), (100, 399)):
        refused(params=[buf[a:a + 300], buf[b:b + 300]])
        refused(exp_avgs=[codes[a:a + 300], codes[b:b + 300]])
        refused(exp_avgs=[codes[a:a + 300], torch.zeros_like(codes[:300])], exp_avg_sqs=[torch.zeros_like(codes[:300]), codes[b:b + 300]])
        refused(params=[buf[a:a + 300], torch.zeros(300)], grads=[torch.zeros(300), buf[b:b + 300]])
    refused(params=[buf[100:400], torch.zeros(300)], grads=[buf[:101], torch.zeros(300)], match="elements")
    steps = torch.zeros(2, dtype=torch.int32)
    refused(steps=[steps[0], steps[0]])
    refused(steps=buf[:2].view(torch.int32), params=[buf[1:301], torch.zeros(300)])
    refused(norm=buf[7], params=[buf[:300], torch.zeros(300)])
    if bits == 8:
        refused(exp_avg_scales=[buf[:2], buf[1:3]])
        refused(exp_avg_scales=[buf[:2], buf[2:4]], exp_avg_sq_scales=[buf[4:6], buf[3:5]])
    # side by side in one buffer, and one gradient for two tensors, are as good as any: only a GPU is missing
    refused(match="CUDA", params=[buf[:300], buf[300:600]], grads=[buf[600:900]] * 2, steps=[steps[0], steps[1]], norm=buf[999])


def test_the_c_entry_refuses():
    import ctypes
    import train_abi as A
    lib = A.library()
    t = (A.AdamwTensor * 1)(A.AdamwTensor(4096, 4096, 4096, 4096, None, None, None, 4096, 10))
    good = dict(lr=1e-3, beta1=0.9, beta2=0.9, eps=1e-8, weight_decay=0.0, state_bits=32, dtype=1, scratch=4096)
    assert lib.tcpxb_adamw_step(t, 1, None, None) == -1 and lib.tcpxb_adamw_step(None, 1, ctypes.byref(A.Adamw(**good)), None) == -1
    for kw in ({"state_bits": 16}, {"dtype": 9}, {"scratch": None}, {"state_bits": 8}, {"compute_norm": 1}):
        assert lib.tcpxb_adamw_step(t, 1, ctypes.byref(A.Adamw(**{**good, **kw})), None) == -1
    for field, x in (("p", None), ("g", None), ("m", None), ("step", None), ("n", -1)):
        u = (A.AdamwTensor * 1)(A.AdamwTensor(4096, 4096, 4096, 4096, None, None, None, 4096, 10))
        setattr(u[0], field, x)
        assert lib.tcpxb_adamw_step(u, 1, ctypes.byref(A.Adamw(**good)), None) == -1, field
    assert lib.tcpxb_grad_norm(t, 1, 1, 0, None, 4096, None) == -1
