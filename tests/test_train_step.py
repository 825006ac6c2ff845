"""The optimizer, and the operators together as a training step uses them."""
import copy
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import train_oracle as oracle
from conftest import free_port
from nccl_plugin_gpudirecttcpx_b200 import ops
from nccl_plugin_gpudirecttcpx_b200.models import LlamaConfig, LlamaDecoder

gpu = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
BF16, F32 = torch.bfloat16, torch.float32


def parameters(dtype=F32, seed=0, sizes=((40, 30), (7,), (300, 5), ())):
    g = torch.Generator("cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, device="cuda", generator=g).to(dtype)) for s in sizes]


def gradients(ps, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, device="cuda", generator=g).to(p.dtype)


@gpu
def test_optimizer_follows_the_formula_with_groups_and_missing_gradients():
    ps = parameters()
    opt = ops.AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.0}], lr=3e-3, weight_decay=0.1)
    want = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64), torch.zeros_like(p, dtype=torch.float64), 0) for p in ps]
    for k in range(4):
        gradients(ps, k)
        if k == 2:
            ps[0].grad = ps[3].grad = None
        opt.step()
        for i, p in enumerate(ps):
            w, m, v, t = want[i]
            if p.grad is not None:
                lr, wd = (1e-2, 0.1) if i < 2 else (3e-3, 0.0)
                want[i] = (*oracle.adamw(w, p.grad, m, v, t + 1, lr, (0.9, 0.999), 1e-8, wd), t + 1)
    for p, (w, _, _, t) in zip(ps, want):
        # a weight is off by its own rounding in each of four steps and the step's few 32-bit roundings (each step is about lr)
        oracle.close(p.detach(), (w, 4 * (4 * oracle.F32 * w.abs() + 40 * oracle.F32 * 1e-2)), "weight")
        assert opt.state[p]["step"] == t


@gpu
@pytest.mark.parametrize("kinds", [(F32, F32), (F32, BF16)])
def test_optimizer_clips_by_the_norm_over_all_groups(kinds):
    ps = [q for n, kind in enumerate(kinds) for q in parameters(kind, n)]
    gradients(ps, 1)
    exact = sum(float(p.grad.double().square().sum()) for p in ps) ** 0.5
    grads = [p.grad.clone() for p in ps]
    before = [p.detach().clone() for p in ps]
    opt = ops.AdamW([{"params": ps[:3]}, {"params": ps[3:]}], max_grad_norm=0.5, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, lr=1.0)
    opt.step()
    assert abs(opt.grad_norm.item() - exact) <= 1e-6 * exact
    for p, g, old in zip(ps, grads, before):
        assert torch.equal(p.grad, g)
        c = g.double() * min(1.0, 0.5 / (exact + 1e-6))
        want = old.double() - c / (c.abs() + 1)
        oracle.close(p.detach(), (want, (oracle.half(p.dtype) if p.dtype == BF16 else 0) * want.abs() + 1e-6), "weight")


@gpu
@pytest.mark.parametrize("bits,master", [(32, False), (8, False), (32, True), (8, True)])
def test_optimizer_state_goes_through_a_state_dict(bits, master, tmp_path):
    ps, qs = parameters(BF16), parameters(BF16)
    make = lambda x: ops.AdamW(x, lr=1e-2, state_bits=bits, master_weights=master, max_grad_norm=1.0)  # noqa: E731
    a, b = make(ps), make(qs)
    for k in range(3):
        gradients(ps, k)
        a.step()
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    b.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    twin = copy.deepcopy(a)
    assert twin.state_bits == bits and twin.max_grad_norm == 1.0
    for p, q in zip(ps, qs):
        assert {n: t.dtype for n, t in a.state[p].items()} == {n: t.dtype for n, t in b.state[q].items()}
    for k in range(2):
        gradients(ps, 10 + k)
        gradients(qs, 10 + k)
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for n, t in a.state[p].items():
            assert torch.equal(t.view(torch.uint8) if t.dim() else t, b.state[q][n].view(torch.uint8) if t.dim() else b.state[q][n])
    with pytest.raises(ValueError):
        ops.AdamW(qs, state_bits=40 - bits, master_weights=master).load_state_dict(a.state_dict())


@gpu
def test_optimizer_in_a_graph_and_on_gradients_of_a_bucket():
    """Gradients are views into one buffer, as data-parallel buckets leave them; the step is captured after a first one."""
    ps = parameters(BF16, sizes=((33, 7), (5,), (64, 64)))
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    bucket = torch.randn(sum(p.numel() for p in ps), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(BF16)
    for p, q, g in zip(ps, qs, bucket.split([p.numel() for p in ps])):
        p.grad, q.grad = g.view(p.shape), g.view(p.shape).clone()
    a, b = ops.AdamW(ps, lr=1e-2, max_grad_norm=1.0), ops.AdamW(qs, lr=1e-2, max_grad_norm=1.0)
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            a.step()
    assert not any(a.state[p] for p in ps)
    a.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    g.replay()
    g.replay()
    for _ in range(3):
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and a.state[p]["step"] == 3


@gpu
def test_norm_rotation_and_attention_together():
    """One layer's chain through autograd, out of a fused projection, is the chain of the single calls."""
    g = torch.Generator("cuda").manual_seed(0)
    b, s, h, hk, d = 2, 300, 8, 2, 64
    qkv = torch.randn(b, s, h + 2 * hk, d, device="cuda", generator=g).to(BF16).requires_grad_()
    wq, wk = (torch.randn(d, device="cuda", generator=g).to(BF16).requires_grad_() for _ in range(2))
    angle = torch.outer(torch.arange(s, device="cuda"), 1e4 ** (-torch.arange(0, d, 2, device="cuda") / d))
    cos, sin = angle.cos(), angle.sin()
    lens = torch.tensor([300, 171], dtype=torch.int32, device="cuda")
    dout = torch.randn(b, s, h, d, device="cuda", generator=g).to(BF16)
    q, k, v = qkv.split((h, hk, hk), 2)
    q2, k2 = ops.qk_norm_rope(q, k, cos, sin, wq, wk)
    out = ops.attention(q2, k2, v, causal=True, key_lengths=lens)
    got = torch.autograd.grad(out, (qkv, wq, wk), dout)
    q, k, v = qkv.detach().split((h, hk, hk), 2)
    wq, wk = wq.detach(), wk.detach()
    q2, k2 = ops.qk_norm_rope(q, k, cos, sin, wq, wk)
    how = {"causal": True, "key_lengths": lens}
    raw, lse = ops.attention_forward(q2, k2, v, **how)
    dq, dk, dv = ops.attention_backward(dout, q2, k2, v, raw, lse, **how)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dq, dk, q, k, cos, sin, wq, wk)
    assert torch.equal(out, raw)
    for x, y in zip(got, (torch.cat((dq, dk, dv), 2), dwq, dwk)):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 256)])
def test_model_gradients(qk_norm, heads):
    """The decoder on the kernels against the decoder in 64 bits.  The plain decoder in the same type rounds at least where
    the kernels do (and its rotation's tables and every step in between besides), so the kernels' gradients are at most as
    far off as twice its; twice, because two roundings of one size can add up where another pair cancels."""
    h, hk, dim = heads
    cfg = LlamaConfig(vocab_size=300, d_model=dim, n_layers=2, n_heads=h, n_kv_heads=hk, ffn_dim=128, qk_norm=qk_norm)
    torch.manual_seed(1)
    exact = LlamaDecoder(cfg).cuda().to(BF16)
    plain, kernels = copy.deepcopy(exact), LlamaDecoder(LlamaConfig(**{**cfg.__dict__, "kernels": True})).cuda().to(BF16)
    kernels.load_state_dict(plain.state_dict())
    exact = exact.double()
    tokens = torch.randint(0, 300, (2, 77), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    grads = []
    for model in (exact, plain, kernels):
        model(tokens[:, :-1], tokens[:, 1:]).backward()
        grads.append({n: p.grad.double() for n, p in model.named_parameters()})
    for n, want in grads[0].items():
        off = [(g[n] - want).norm() / want.norm() for g in grads[1:]]
        assert off[1] <= 2 * off[0], (n, off)


@gpu
@pytest.mark.parametrize("qk_norm", [False, True])
def test_model_under_autocast(qk_norm):
    """32-bit parameters, heads in 16 bits.  Against the decoder in 64 bits, as in test_model_gradients; the norms' weights are
    numbers that 16 bits hold, so that their cast takes nothing the plain decoder keeps."""
    cfg = LlamaConfig(vocab_size=300, d_model=64, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=128, qk_norm=qk_norm)
    torch.manual_seed(5)
    plain = LlamaDecoder(cfg).cuda()
    with torch.no_grad():
        for n, p in plain.named_parameters():
            if n.endswith(("q_norm.weight", "k_norm.weight")):
                p.copy_((1 + 0.2 * torch.randn_like(p)).to(BF16))
    exact, kernels = copy.deepcopy(plain).double(), LlamaDecoder(LlamaConfig(**{**cfg.__dict__, "kernels": True})).cuda()
    kernels.load_state_dict(plain.state_dict())
    tokens = torch.randint(0, 300, (2, 77), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    grads = []
    for model in (exact, plain, kernels):
        with torch.autocast("cuda", BF16, enabled=model is not exact):
            loss = model(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        grads.append({n: p.grad.double() for n, p in model.named_parameters()})
    for n, want in grads[0].items():
        off = [(g[n] - want).norm() / want.norm() for g in grads[1:]]
        assert off[1] <= 2 * off[0], (n, off)


@gpu
def test_a_captured_step_of_the_model():
    """Forward, backward and optimizer in one graph give what eager steps give."""
    cfg = LlamaConfig.tiny()
    cfg.qk_norm = cfg.kernels = True
    torch.manual_seed(3)
    eager = LlamaDecoder(cfg).cuda().to(BF16)
    graph = copy.deepcopy(eager)
    tokens = torch.randint(0, cfg.vocab_size, (2, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(4))

    def step(model, opt):
        grads = torch.autograd.grad(model(tokens[:, :-1], tokens[:, 1:]), list(model.parameters()))
        for p, g in zip(model.parameters(), grads):
            p.grad = g
        opt.step()

    a, b = (ops.AdamW(m.parameters(), lr=1e-3, max_grad_norm=1.0, state_bits=8) for m in (eager, graph))
    for _ in range(4):
        step(eager, a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graph, b)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(graph, b)
    for _ in range(3):
        g.replay()
    for p, q in zip(eager.parameters(), graph.parameters()):
        assert torch.equal(p, q)


@gpu
def test_other_threads_run_while_a_launch_waits():
    """A full queue of launches makes the next one wait; a second Python thread goes on meanwhile."""
    import threading
    import time
    q = torch.randn(1, 64, 2, 64, device="cuda").to(BF16)
    p, g, m, v = (torch.zeros(10, device="cuda") for _ in range(4))
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    cos = sin = torch.zeros(64, 32, device="cuda")
    for call in (lambda: ops.attention(q, q, q), lambda: ops.qk_norm_rope(q, q, cos, sin), lambda: ops.adamw_step([p], [g], [m], [v], steps, lr=0.0)):
        call()
        torch.cuda.synchronize()
        ticks, done = [], threading.Event()

        def tick():
            while not done.is_set():
                ticks.append(time.perf_counter())
                time.sleep(0.002)

        thread = threading.Thread(target=tick)
        thread.start()
        try:
            torch.cuda._sleep(1_500_000_000)  # most of a second
            began = time.perf_counter()
            for _ in range(3000):
                call()
            waited = time.perf_counter() - began
        finally:
            done.set()
            thread.join()
        torch.cuda.synchronize()
        assert waited > 0.4  # the queue was full
        assert max(b - a for a, b in zip(ticks, ticks[1:])) < waited / 2


def _ddp(args):
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=1", "--master-addr", "127.0.0.1", "--master-port", str(free_port()),
           "-m", "nccl_plugin_gpudirecttcpx_b200.parallel.ddp", "--tiny", "--steps", "3", "--warmup", "2", *args]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=240, cwd=str(ROOT), env={**os.environ, "PYTHONPATH": str(ROOT)})
    return r, [json.loads(line) for line in r.stdout.splitlines() if line.startswith('{"bench"')]


@gpu
@pytest.mark.parametrize("args", [["--qk-norm"], ["--state-bits", "8", "--max-grad-norm", "1.0"]])
def test_the_ddp_command_runs_on_the_kernels(args):
    r, rows = _ddp(["--transport", "engine", "--kernels", "--nics", "2", "--nthreads", "2", *args])
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert len(rows) == 1 and rows[0]["kernels"] and rows[0]["replicas_in_sync"] and rows[0]["engine_buckets"] > 0


def test_the_ddp_command_refuses_kernels_without_gpus():
    from nccl_plugin_gpudirecttcpx_b200.parallel.ddp import parse_args
    for args in (["--kernels", "--backend", "gloo"], ["--state-bits", "8"], ["--max-grad-norm", "1.0"]):
        with pytest.raises(SystemExit):
            parse_args(args)


def test_model_with_head_norms_on_the_cpu():
    cfg = LlamaConfig.tiny()
    cfg.qk_norm = True
    m = LlamaDecoder(cfg)
    tok = torch.randint(0, cfg.vocab_size, (2, 16))
    m(tok, tok).backward()
    assert all(p.grad is not None for p in m.parameters())
    assert sum(n.endswith(("q_norm.weight", "k_norm.weight")) for n, _ in m.named_parameters()) == 2 * cfg.n_layers


def test_a_refused_group_is_not_kept():
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    opt = ops.AdamW([p], lr=0.5)
    for kind, kw in ((ValueError, {"lr": -1.0}), (TypeError, {"lr": torch.tensor(0.1)}), (ValueError, {"betas": (1.0, 0.9)})):
        with pytest.raises(kind):
            opt.add_param_group({"params": [q], **kw})
        assert [g["lr"] for g in opt.param_groups] == [0.5]
    opt.add_param_group({"params": [q]})
    assert len(opt.param_groups) == 2


def test_states_of_another_optimizer_are_refused():
    """torch.optim.AdamW's have the same names and other types; nothing is loaded of what is refused."""
    p, q = torch.nn.Parameter(torch.zeros(300)), torch.nn.Parameter(torch.zeros(300))
    other = torch.optim.AdamW([p])
    p.grad = torch.ones(300)
    other.step()
    good = {"step": torch.ones((), dtype=torch.int32), "exp_avg": torch.ones(300), "exp_avg_sq": torch.ones(300)}
    opt = ops.AdamW([q])
    groups = opt.state_dict()["param_groups"]
    opt.load_state_dict({"state": {0: good}, "param_groups": groups})
    bad = [other.state_dict()["state"][0]] + [{**good, n: t} for n, t in (
        ("step", torch.ones(2, dtype=torch.int32)), ("exp_avg", torch.ones(299)), ("exp_avg", torch.ones(300, dtype=BF16)), ("exp_avg_sq", torch.ones(300, 2)[:, 0]))]
    for state in bad:
        with pytest.raises(ValueError, match="state"):
            opt.load_state_dict({"state": {0: state}, "param_groups": groups})
        assert all(torch.equal(opt.state[q][n], t) and opt.state[q][n].dtype is t.dtype for n, t in good.items())
    small = {n: torch.ones(1 if n == "step" else 2 if n.endswith("scale") else 300).to(torch.int32 if n == "step" else torch.float32 if n.endswith("scale") else torch.float8_e4m3fn)
             for n in ("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
    opt = ops.AdamW([q], state_bits=8)
    opt.load_state_dict({"state": {0: small}, "param_groups": groups})
    for n, t in (("exp_avg", torch.ones(300)), ("exp_avg_scale", torch.ones(300))):
        with pytest.raises(ValueError, match="state"):
            opt.load_state_dict({"state": {0: {**small, n: t}}, "param_groups": groups})


def test_the_norm_of_a_step_without_gradients_is_zero():
    p = torch.nn.Parameter(torch.zeros(3))
    opt = ops.AdamW([{"params": []}, {"params": [p]}], max_grad_norm=1.0)
    opt.grad_norm = torch.tensor(7.0)  # an earlier step's
    opt.step()
    assert opt.grad_norm.item() == 0.0
    assert not opt.state


def test_optimizer_clips_over_several_devices(monkeypatch):
    """One norm over all devices, given to each on its own; the kernels' calls are recorded, the second device has no memory."""
    from nccl_plugin_gpudirecttcpx_b200.ops import optimizer
    norms, calls = {"cpu": 3.0, "meta": 4.0}, []
    # a device without memory cannot give its norm away: both come from the first one's
    monkeypatch.setattr(optimizer, "grad_norm", lambda grads: torch.tensor(norms[grads[0].device.type]))
    monkeypatch.setattr(optimizer, "adamw_step", lambda ps, *args, norm, **kw: calls.append((ps[0].device, norm)))
    ps = [torch.nn.Parameter(torch.zeros(3, device=d)) for d in ("cpu", "meta")]
    for p in ps:
        p.grad = torch.zeros_like(p)
    opt = ops.AdamW(ps, max_grad_norm=1.0)
    opt.step()
    assert [d.type for d, _ in calls] == [n.device.type for _, n in calls] == ["cpu", "meta"]
    assert calls[0][1].item() == 5.0 and opt.grad_norm.item() == 5.0


def test_optimizer_refusals():
    p = torch.nn.Parameter(torch.zeros(3))
    for kind, kw in ((ValueError, {"lr": -1.0}), (ValueError, {"betas": (1.0, 0.9)}), (ValueError, {"eps": -1.0}), (ValueError, {"weight_decay": -1.0}),
                     (ValueError, {"state_bits": 16}), (ValueError, {"max_grad_norm": -1.0}), (TypeError, {"lr": torch.tensor(0.1)})):
        with pytest.raises(kind):
            ops.AdamW([p], **kw)
    with pytest.raises(TypeError):
        ops.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    with pytest.raises(ValueError):
        ops.AdamW([torch.nn.Parameter(torch.zeros(3, 4).t())])
    opt = ops.AdamW([p])
    p.grad = torch.zeros(3)
    with pytest.raises(ValueError):  # not on a GPU
        opt.step()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_is_refused(device):
    """A dual tensor requires no gradient; its tangent is not dropped without a word, through `make_dual` or `torch.func.jvp`."""
    import torch.autograd.forward_ad as fwd
    q, k, v = (torch.randn(1, 6, 2, 16, device=device).to(BF16) for _ in range(3))
    cos, sin = torch.randn(6, 8, device=device), torch.randn(6, 8, device=device)
    w = torch.ones(16, device=device, dtype=BF16)
    lse = torch.zeros(1, 2, 6, device=device)
    calls = [(lambda x: ops.attention(x, k, v), q), (lambda x: ops.attention(q, x, v), k), (lambda x: ops.attention(q, k, x), v),
             (lambda x: ops.attention_forward(x, k, v)[0], q), (lambda x: ops.attention_backward(x, q, k, v, q, lse)[0], q),
             (lambda x: ops.qk_norm_rope(x, k, cos, sin)[0], q), (lambda x: ops.qk_norm_rope(q, k, x, sin)[0], cos),
             (lambda x: ops.qk_norm_rope(q, k, cos, sin, x, w)[0], w), (lambda x: ops.qk_norm_rope_backward(x, k, q, k, cos, sin)[0], q)]
    for call, x in calls:
        with fwd.dual_level():
            # autograd's own refusal, of a tensor that has both, comes behind the forward pass
            for y in (x,) if device == "cpu" else (x, x.clone().requires_grad_()):
                with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp"):
                    call(fwd.make_dual(y, torch.ones_like(x)))
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
