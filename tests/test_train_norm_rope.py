"""Head norms with rotation, forward and backward, against the definition in 64 bits."""
import math

import pytest
import torch

import train_oracle as oracle
from nccl_plugin_gpudirecttcpx_b200 import ops

gpu = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(b, s, h, hk, d, dtype, norm, seed=0, positions=None, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=device, generator=g).to(dtype)

    angle = torch.arange(positions or s, device=device, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, d, 2, device=device) / d)
    w = (normal(d), normal(d)) if norm else (None, None)
    return [normal(b, s, h, d), normal(b, s, hk, d), angle.cos().float(), angle.sin().float(), *w], [normal(b, s, h, d), normal(b, s, hk, d)]


def check(x, dy, eps=1e-5, positions=None):
    q, k, cos, sin, wq, wk = x
    outs = ops.qk_norm_rope(*x, eps=eps, positions=positions)
    grads = ops.qk_norm_rope_backward(*dy, *x, eps=eps, positions=positions)
    for n, (t, w) in enumerate(((q, wq), (k, wk))):
        want = oracle.norm_rope(t, w, cos, sin, dy[n], eps, positions)
        oracle.close(outs[n], want["y"], "y")
        oracle.close(grads[n], want["dx"], "dx")
        if w is None:
            assert grads[2 + n] is None
        else:
            oracle.close(grads[2 + n], want["dw"], "dw")
    return (*outs, *grads)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("b,s,h,hk,d", [(1, 1, 1, 1, 8), (2, 3, 4, 2, 16), (1, 65, 3, 1, 24), (3, 33, 5, 5, 64), (2, 257, 32, 8, 64), (1, 100, 4, 2, 80),
                                        (2, 77, 7, 1, 128), (1, 31, 2, 2, 192), (1, 50, 3, 2, 256), (1, 4099, 2, 1, 32)])
def test_against_the_definition(b, s, h, hk, d, norm, dtype):
    check(*inputs(b, s, h, hk, d, dtype, norm, seed=s))


@gpu
@pytest.mark.parametrize("norm", [True, False])
def test_positions(norm):
    x, dy = inputs(2, 50, 4, 2, 64, BF16, norm, seed=1, positions=1000)
    pos = torch.randint(0, 1000, (2, 50), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    pos[0, 0], pos[1, 3] = 999, 0
    check(x, dy, positions=pos)
    check(x, dy, positions=pos.t().contiguous().t())
    same = torch.arange(50, device="cuda").expand(2, 50)
    assert all(torch.equal(a, b) for a, b in zip(check(x, dy), check(x, dy, positions=same)) if a is not None)


@gpu
def test_positions_outside_the_tables_give_nan_there_alone():
    x, dy = inputs(1, 6, 2, 1, 64, BF16, False, seed=2, positions=10)
    pos = torch.tensor([[0, 10, 3, -1, 9, 1 << 40]], device="cuda")
    bad = torch.tensor([False, True, False, True, False, True], device="cuda")
    for t in (*ops.qk_norm_rope(*x, positions=pos), *ops.qk_norm_rope_backward(*dy, *x, positions=pos)[:2]):
        assert t[0, bad].isnan().all() and t[0, ~bad].isfinite().all()


@gpu
def test_rows_of_zeros_and_large_values():
    x, dy = inputs(1, 40, 4, 2, 64, F32, True, seed=3)
    x[0][0, 5], x[1][0, 6] = 0, 0
    x[0][0, 7] *= 1e15
    x[1][0, 8] *= 1e-15
    check(x, dy)
    check(x, dy, eps=1e-30)


@gpu
def test_nan_stays_in_its_row():
    x, _ = inputs(1, 40, 4, 2, 64, BF16, True, seed=4)
    want = ops.qk_norm_rope(*x)
    x[0][0, 11, 2, 5] = math.nan
    got = ops.qk_norm_rope(*x)
    assert got[0][0, 11, 2].isnan().all() and torch.equal(got[1], want[1])
    got[0][0, 11, 2] = want[0][0, 11, 2]
    assert torch.equal(got[0], want[0])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_and_copies(dtype):
    """A fused projection, heads first, odd offsets: the same bits."""
    x, dy = inputs(2, 60, 4, 2, 64, dtype, True, seed=5)
    q, k, *rest = x
    want = check(x, dy)
    fused = torch.cat((q, k, k), 2)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    first = q.transpose(1, 2).contiguous().transpose(1, 2)
    w2 = torch.empty(65, dtype=dtype, device="cuda")[1:].copy_(rest[2])
    for q2, k2 in ((fused[:, :, :4], fused[:, :, 4:6]), (odd, k), (first, k)):
        got = check([q2, k2, rest[0], rest[1], w2, rest[3]], [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dy])
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
@pytest.mark.parametrize("norm", [True, False])
def test_autograd_and_differences(norm):
    x, dy = inputs(2, 20, 4, 2, 32, F32, norm, seed=6)
    leaves = [t if n in (2, 3) or t is None else t.clone().requires_grad_() for n, t in enumerate(x)]
    outs = ops.qk_norm_rope(*leaves)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    got = torch.autograd.grad(outs, wanted, dy)
    raw = [t for t in ops.qk_norm_rope_backward(*dy, *x) if t is not None]
    assert all(torch.equal(a, b) for a, b in zip(got, raw))
    step = 2.0 ** -10
    for n, grad in zip([i for i in (0, 1, 4, 5) if x[i] is not None], got):
        way = torch.randn(grad.shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(n))

        def value(t):
            total = 0.0
            y = [None if v is None else v.double() for v in x]
            y[n] = y[n] + t * way
            for i in (0, 1):
                h = y[i] if not norm else y[i] * (y[i].square().mean(-1, keepdim=True) + 1e-6).rsqrt() * y[4 + i]
                total = total + (oracle.rotate(h, y[2][:, None], y[3][:, None]) * dy[i].double()).sum()
            return total

        diff = (value(step) - value(-step)) / (2 * step)
        room = 2.0 ** -14 * (grad.double() * way).abs().sum()  # 32-bit sums of up to 160 rows and 64 products, and the difference's step^2
        assert abs((grad.double() * way).sum() - diff) <= room


@gpu
def test_one_output_unused():
    x, dy = inputs(1, 20, 4, 2, 64, BF16, True, seed=7)
    q, w = x[0].clone().requires_grad_(), x[4].clone().requires_grad_()
    ops.qk_norm_rope(q, x[1], x[2], x[3], w, x[5])[0].backward(dy[0])
    raw = ops.qk_norm_rope_backward(dy[0], torch.zeros_like(dy[1]), *x)
    assert torch.equal(q.grad, raw[0]) and torch.equal(w.grad, raw[2])


@gpu
def test_same_bits_every_time_and_in_a_graph():
    x, dy = inputs(2, 500, 16, 4, 64, BF16, True, seed=8)
    first = check(x, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, check(x, dy)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = (*ops.qk_norm_rope(*x, eps=1e-5), *ops.qk_norm_rope_backward(*dy, *x, eps=1e-5))
    fresh, fresh_dy = inputs(2, 500, 16, 4, 64, BF16, True, seed=9)
    for a, b in zip(x + dy, fresh + fresh_dy):
        a.copy_(b)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, check(x, dy)))


@gpu
@pytest.mark.parametrize("b,s", [(0, 5), (2, 0)])
def test_nothing_to_do(b, s):
    x, dy = inputs(b, s, 4, 2, 64, BF16, True)
    outs, grads = ops.qk_norm_rope(*x), ops.qk_norm_rope_backward(*dy, *x)
    assert outs[0].shape == x[0].shape and not grads[2].any() and not grads[3].any()


def test_refusals():
    x, dy = inputs(2, 5, 4, 2, 64, BF16, True, device="cpu")
    q, k, cos, sin, wq, wk = x
    pos = torch.zeros(2, 5, dtype=torch.int64)
    bad = [
        (ValueError, lambda: ops.qk_norm_rope(q[0], k, cos, sin)),
        (TypeError, lambda: ops.qk_norm_rope(q, k.float(), cos, sin)),
        (TypeError, lambda: ops.qk_norm_rope(q.double(), k.double(), cos, sin)),
        (ValueError, lambda: ops.qk_norm_rope(q, k[:, :4], cos, sin)),
        (ValueError, lambda: ops.qk_norm_rope(q[..., :60], k[..., :60], cos, sin)),
        (TypeError, lambda: ops.qk_norm_rope(q, k, cos.bfloat16(), sin)),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos[:4], sin[:4])),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos[:, :16], sin[:, :16])),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin, wq)),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin, wq[:32], wk)),
        (TypeError, lambda: ops.qk_norm_rope(q, k, cos, sin, wq.float(), wk.float())),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin, eps=-1.0)),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin, eps=math.nan)),
        (TypeError, lambda: ops.qk_norm_rope(q, k, cos, sin, positions=pos.int())),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin, positions=pos[:1])),
        (ValueError, lambda: ops.qk_norm_rope(q, k, cos, sin)),  # not on a GPU
        (ValueError, lambda: ops.qk_norm_rope_backward(dy[0][:1], dy[1], q, k, cos, sin)),
        (TypeError, lambda: ops.qk_norm_rope_backward(dy[0], dy[1].float(), q, k, cos, sin)),
        (ValueError, lambda: ops.qk_norm_rope_backward(*dy, q, k, cos, sin)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_the_c_entry_refuses():
    import ctypes
    import train_abi as A
    lib = A.library()
    assert lib.tcpxb_norm_rope_forward(None, None) == -1

    def args(**kw):
        a = A.NormRope(b=1, s=4, heads=4, kv_heads=2, d=64, positions=4, eps=1e-6, dtype=1, q=4096, k=4096, q_s=256, k_s=256, q_h=64, k_h=64, cos=4096, sin=4096, q_out=4096, k_out=4096)
        for n, x in kw.items():
            setattr(a, n, x)
        return ctypes.byref(a)

    for kw in ({"b": -1}, {"heads": 0}, {"d": 60}, {"d": 264}, {"dtype": 0}, {"positions": 3}, {"cos": 0}, {"wq": 4096}, {"q_out": 0},
               {"q": 4098}, {"k_s": 1}, {"cos": 4100}, {"b": 1 << 30}):
        assert lib.tcpxb_norm_rope_forward(args(**kw), None) == -1, kw
    assert lib.tcpxb_norm_rope_backward(args(), None) == -1
