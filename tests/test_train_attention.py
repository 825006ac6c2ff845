"""Attention forward and backward against the definition in 64 bits, at the sizes and masks where tiles end."""
import math

import pytest
import torch

import train_oracle as oracle
from nccl_plugin_gpudirecttcpx_b200 import _build, ops

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def inputs(b, sq, sk, h, hk, d, dtype, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn(s, device=device, generator=g).to(dtype) for s in ((b, sq, h, d), (b, sk, hk, d), (b, sk, hk, d), (b, sq, h, d))]


def check(q, k, v, dout, causal=False, lengths=None, scale=None):
    how = {"causal": causal, "key_lengths": lengths, "scale": scale}
    out, lse = ops.attention_forward(q, k, v, **how)
    dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, **how)
    want = oracle.attention(q, k, v, dout, causal, lengths, scale)
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        oracle.close(got, want[name], name)
    return out, lse, dq, dk, dv


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,sq,sk,h,hk,d", [
    (1, 1, 1, 1, 1, 8), (2, 1, 17, 4, 2, 64), (1, 17, 1, 2, 1, 64), (3, 64, 64, 4, 2, 16), (1, 127, 127, 2, 1, 64), (1, 128, 128, 2, 1, 128),
    (1, 129, 129, 2, 2, 64), (1, 129, 127, 2, 2, 128), (1, 200, 72, 3, 1, 40), (2, 257, 513, 6, 3, 96), (1, 300, 641, 4, 4, 64),
    (2, 255, 256, 8, 1, 72), (1, 1000, 1000, 2, 1, 128), (1, 385, 385, 5, 5, 24), (1, 2, 1500, 4, 2, 64), (1, 1500, 3, 4, 2, 120)])
def test_against_the_definition(b, sq, sk, h, hk, d, causal, dtype):
    check(*inputs(b, sq, sk, h, hk, d, dtype, seed=sq * 7 + sk), causal=causal)


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("s,lengths", [(130, [130, 0, 1, 129]), (513, [512, 128, 127, 300]), (64, [64, 63, 100, -5])])
def test_key_lengths(s, lengths, causal):
    """Lengths that end inside and at tiles; none; values beyond the ends count as the nearer end."""
    q, k, v, dout = inputs(4, s, s, 4, 2, 64, BF16, seed=s)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = check(q, k, v, dout, causal, lens)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), s)
        assert not got[3][i, n:].any() and not got[4][i, n:].any()
        if n == 0:
            assert not got[0][i].any() and not got[2][i].any() and (got[1][i] == -math.inf).all()


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_behind_a_length_has_no_influence(bad, d):
    q, k, v, dout = inputs(3, 200, 300, 4, 2, d, BF16, seed=3)
    lens = torch.tensor([300, 150, 0], dtype=torch.int32, device="cuda")
    clean = [t.clone() for t in check(q, k, v, dout, False, lens)]
    for i, n in enumerate(lens.tolist()):
        k[i, n:], v[i, n:] = bad, bad
    for a, b in zip(clean, check(q, k, v, dout, False, lens)):
        assert torch.equal(a, b)


@gpu
def test_nan_of_a_query_stays_in_its_row():
    q, k, v, dout = inputs(1, 200, 200, 2, 2, 64, BF16, seed=4)
    want = ops.attention_forward(q, k, v)[0]
    q[0, 77, 1] = math.nan
    got = ops.attention_forward(q, k, v)[0]
    assert got[0, 77, 1].isnan().all()
    got[0, 77, 1] = want[0, 77, 1]
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("factor", [1e-3, 30.0])
def test_flat_and_peaked_rows(factor):
    """Scores of almost one size, and scores of hundreds whose exponentials span the range."""
    q, k, v, dout = inputs(1, 300, 300, 2, 1, 64, BF16, seed=5)
    check((q * factor).to(BF16), k, v, dout, True)


@gpu
def test_scores_that_fall_and_rise_along_the_keys():
    """The running maximum changes in every tile, or never after the first."""
    q, k, v, dout = inputs(1, 64, 1024, 1, 1, 64, BF16, seed=6)
    q[..., 0] = 8.0
    ramp = torch.linspace(-16, 16, 1024, device="cuda")
    for sign in (1, -1):
        k[0, :, 0, 0] = (sign * ramp).to(BF16)
        check(q, k, v, dout)


@gpu
def test_scale():
    q, k, v, dout = inputs(1, 150, 150, 2, 1, 64, F16, seed=7)
    check(q, k, v, dout, True, scale=0.31)


@gpu
def test_views_and_copies():
    """Heads first, a fused projection, odd offsets that have to be copied, a broadcast batch: the same bits."""
    q, k, v, dout = inputs(2, 150, 150, 4, 2, 64, BF16, seed=8)
    want = check(q, k, v, dout, True)
    fused = torch.cat((q, k, v), 2)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape).copy_(q)
    wide = torch.empty(2, 150, 4, 65, dtype=BF16, device="cuda")[..., :64].copy_(q)
    every_second = torch.empty(2, 150, 4, 128, dtype=BF16, device="cuda")[..., ::2].copy_(q)
    first = q.transpose(1, 2).contiguous().transpose(1, 2)
    for q2, (k2, v2) in [(x, (k, v)) for x in (odd, wide, every_second, first)] + [(fused[:, :, :4], (fused[:, :, 4:6], fused[:, :, 6:]))]:
        out, lse = ops.attention_forward(q2, k2, v2, causal=True)
        grads = ops.attention_backward(dout.transpose(1, 2).contiguous().transpose(1, 2), q2, k2, v2, out, lse, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(want, (out, lse, *grads)))
    one = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    check(q, *one, dout, True)


@gpu
def test_same_bits_every_time():
    q, k, v, dout = inputs(2, 700, 700, 8, 2, 64, BF16, seed=9)
    first = check(q, k, v, dout, True)
    out, lse = ops.attention_forward(q, k, v, causal=True)
    for _ in range(5):
        again = (*ops.attention_forward(q, k, v, causal=True), *ops.attention_backward(dout, q, k, v, out, lse, causal=True))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@gpu
def test_autograd_and_differences():
    """Gradients through autograd are the backward call's, and agree with central differences of the definition."""
    q, k, v, dout = inputs(1, 70, 70, 4, 2, 64, BF16, seed=10)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, causal=True)
    got = torch.autograd.grad(out, leaves, dout)
    raw = ops.attention_forward(q, k, v, causal=True)
    assert torch.equal(out, raw[0])
    assert all(torch.equal(a, b) for a, b in zip(got, ops.attention_backward(dout, q, k, v, *raw, causal=True)))
    want = oracle.attention(q, k, v, dout, True)
    step = 2.0 ** -12
    for n, (name, grad) in enumerate(zip(("dq", "dk", "dv"), got)):
        way = torch.randn(grad.shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(n))

        def value(t):
            x = [q.double(), k.double(), v.double()]
            x[n] = x[n] + t * way
            x = [y.transpose(1, 2) for y in x]
            x[1:] = [y.repeat_interleave(2, 1) for y in x[1:]]
            s = (x[0] @ x[1].mT * 64 ** -0.5).masked_fill(~oracle.visible(1, 70, 70, True, None).cuda(), -torch.inf)
            return ((s.softmax(-1) @ x[2]).transpose(1, 2) * dout.double()).sum()

        diff = (value(step) - value(-step)) / (2 * step)
        # the difference's own error: a third derivative times step^2 / 6, below 2^-24 of the sum of magnitudes times a hundred
        room = (want[name][1] * way.abs()).sum() + 100 * step ** 2 * (grad.double() * way).abs().sum()
        assert abs((grad.double() * way).sum() - diff) <= room
    with torch.no_grad():
        assert not ops.attention(*leaves, causal=True).requires_grad


@gpu
def test_gradients_where_only_some_are_wanted():
    q, k, v, dout = inputs(1, 33, 33, 2, 2, 64, BF16, seed=11)
    v2 = v.clone().requires_grad_()
    ops.attention(q, k, v2).backward(dout)
    out, lse = ops.attention_forward(q, k, v)
    assert torch.equal(v2.grad, ops.attention_backward(dout, q, k, v, out, lse)[2])


@gpu
def test_status_stays_zero():
    status = ops.status_buffer()
    q, k, v, dout = inputs(2, 300, 300, 8, 2, 64, BF16, seed=13)
    out, lse = ops.attention_forward(q, k, v, causal=True, status=status)
    ops.attention_backward(dout, q, k, v, out, lse, causal=True, status=status)
    assert not status.any()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal", [
    (1, 1, 1, 1, 1, 8, False), (2, 300, 300, 4, 2, 64, True), (2, 300, 300, 4, 2, 128, True), (1, 40, 3000, 2, 1, 64, False), (1, 40, 3000, 2, 1, 128, True),
    (1, 700, 20, 8, 1, 40, False), (16, 513, 513, 8, 2, 64, True), (3, 150, 90, 4, 4, 96, True)])
def test_void_outputs_are_nan(b, sq, sk, h, hk, d, causal, dtype):
    """A status that tells of a wait that ran out makes what follows void: no work, NaN wherever a row sees something, the status
    kept.  Blocks alone and in clusters, rows that see nothing, ends of tiles; with the status cleared all is as before."""
    q, k, v, dout = inputs(b, sq, sk, h, hk, d, dtype, seed=14)
    status = ops.status_buffer()
    out, lse = ops.attention_forward(q, k, v, causal=causal, status=status)
    want = out, lse, *ops.attention_backward(dout, q, k, v, out, lse, causal=causal, status=status)
    kept = [t.clone() for t in (q, k, v, dout, out, lse)]
    assert not status.any()
    status[0] = 3
    got = *ops.attention_forward(q, k, v, causal=causal, status=status), *ops.attention_backward(dout, q, k, v, out, lse, causal=causal, status=status)
    sees = oracle.visible(b, sq, sk, causal, None).any(-1).cuda()  # [b, 1, sq]
    assert got[1].isnan().eq(sees).all() and (got[1][~sees.expand_as(lse)] == -math.inf).all()
    rows = sees.transpose(1, 2)[..., None]
    for x in (got[0], got[2]):
        assert x.isnan().eq(rows).all() and not x[~rows.expand_as(x)].any()
    assert got[3].isnan().all() and got[4].isnan().all()
    assert status.tolist() == [3] + [0] * (status.numel() - 1)
    assert all(torch.equal(x, y) for x, y in zip(kept, (q, k, v, dout, out, lse)))
    status.zero_()
    got = *ops.attention_forward(q, k, v, causal=causal, status=status), *ops.attention_backward(dout, q, k, v, out, lse, causal=causal, status=status)
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and not status.any()


HOLDER = r"""
#include <cstdint>
// Holds an SM's tensor memory for some time, beside whatever else finds room there.
__global__ void hold(unsigned long long ns) {
  __shared__ uint32_t at;
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&at)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  do {
    __nanosleep(100000);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  } while (t - t0 < ns);
  __syncwarp();
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(at) : "memory");
}
extern "C" int run(int blocks, unsigned long long ns, void* stream) {
  const int room = 118 << 10;  // one block on an SM, and room for one of attention's
  if (cudaFuncSetAttribute(hold, cudaFuncAttributeMaxDynamicSharedMemorySize, room)) return 1;
  hold<<<blocks, 32, room, (cudaStream_t)stream>>>(ns);
  return cudaGetLastError();
}
"""


@gpu
@pytest.mark.skipif(not _build._nvcc(), reason="needs nvcc")
def test_tensor_memory_that_another_kernel_holds(tmp_path):
    """Blocks that get their tensor memory later than a wait may last: no wait runs out over it."""
    import ctypes
    import subprocess
    import time
    (tmp_path / "hold.cu").write_text(HOLDER)
    subprocess.run([_build._nvcc(), *_build.NVCC_ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", tmp_path / "hold.so", tmp_path / "hold.cu"], check=True)
    hold = ctypes.CDLL(str(tmp_path / "hold.so")).run
    hold.argtypes = ctypes.c_int, ctypes.c_uint64, ctypes.c_void_p
    q, k, v, dout = inputs(8, 900, 900, 8, 2, 64, BF16, seed=15)  # rings that wrap
    status = ops.status_buffer()
    out, lse = ops.attention_forward(q, k, v, status=status)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    assert hold(torch.cuda.get_device_properties(0).multi_processor_count, 2_600_000_000, side.cuda_stream) == 0
    time.sleep(0.2)
    began = time.time()
    again = ops.attention_forward(q, k, v, status=status)
    torch.cuda.current_stream().synchronize()
    waited = time.time() - began
    torch.cuda.synchronize()
    assert not status.any() and torch.equal(out, again[0]) and torch.equal(lse, again[1])
    assert waited > 2.1  # else nothing was held


@gpu
@pytest.mark.parametrize("b,sq,sk", [(0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)])
def test_nothing_to_do(b, sq, sk):
    q, k, v, dout = inputs(b, sq, sk, 4, 2, 64, BF16)
    out, lse = ops.attention_forward(q, k, v)
    grads = ops.attention_backward(dout, q, k, v, out, lse)
    assert not out.any() and (lse == -math.inf).all() and not any(g.any() for g in grads)
    assert [g.shape for g in grads] == [q.shape, k.shape, v.shape]


@gpu
def test_on_another_stream_and_in_two_graphs():
    """Captured calls replay on new contents of their inputs; two graphs replay at the same time."""
    sets = [inputs(1, 260, 260, 4, 2, 64, BF16, seed=20 + i) for i in range(2)]
    runs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for s in sets:
        with torch.cuda.stream(side):
            ops.attention_backward(s[3], *s[:3], *ops.attention_forward(*s[:3], causal=True), causal=True)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out, lse = ops.attention_forward(*s[:3], causal=True)
            runs.append((g, (out, lse, *ops.attention_backward(s[3], *s[:3], out, lse, causal=True))))
    for s, fresh in zip(sets, [inputs(1, 260, 260, 4, 2, 64, BF16, seed=30 + i) for i in range(2)]):
        for a, b in zip(s, fresh):
            a.copy_(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(3):
        for (g, _), st in zip(runs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, (_, got) in zip(sets, runs):
        want = check(*s, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_offsets_beyond_32_bits():
    """Batches 2^31 elements and heads 2^30 elements apart in one buffer."""
    buf = torch.empty((1 << 32) + (1 << 20), dtype=BF16, device="cuda")
    q, k, v, dout = inputs(2, 150, 150, 2, 2, 64, BF16, seed=12)
    far = buf.as_strided((2, 150, 2, 64), (1 << 31, 64, 1 << 30, 1))
    want = check(q, k, v, dout, True)
    for n in range(3):
        far.copy_((q, k, v)[n])
        x = [q, k, v]
        x[n] = far
        out, lse = ops.attention_forward(*x, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(want, (out, lse, *ops.attention_backward(dout, *x, out, lse, causal=True))))


def test_refusals():
    q, k, v, dout = inputs(2, 5, 7, 4, 2, 64, BF16, device="cpu")
    bad = [
        (ValueError, lambda: ops.attention(q[0], k, v)),
        (TypeError, lambda: ops.attention(q.float(), k, v)),
        (TypeError, lambda: ops.attention(q, k.half(), v)),
        (TypeError, lambda: ops.attention(q.float(), k.float(), v.float())),
        (ValueError, lambda: ops.attention(q, k, v[:, :6])),
        (ValueError, lambda: ops.attention(q, k[:1], v[:1])),
        (ValueError, lambda: ops.attention(q[:, :, :3], k, v)),
        (ValueError, lambda: ops.attention(q, k[:, :, :0], v[:, :, :0])),
        (ValueError, lambda: ops.attention(q[..., :60], k[..., :60], v[..., :60])),
        (ValueError, lambda: ops.attention(*(torch.zeros(1, 2, 2, 136, dtype=BF16),) * 3)),
        (ValueError, lambda: ops.attention(q, k, v, scale=0.0)),
        (ValueError, lambda: ops.attention(q, k, v, scale=math.nan)),
        (ValueError, lambda: ops.attention(q, k, v, scale=-1.0)),
        (TypeError, lambda: ops.attention(q, k, v, key_lengths=torch.ones(2, dtype=torch.int64))),
        (ValueError, lambda: ops.attention(q, k, v, key_lengths=torch.ones(3, dtype=torch.int32))),
        (ValueError, lambda: ops.attention_forward(q, k, v, status=torch.zeros(4))),
        (ValueError, lambda: ops.attention(q, k, v)),  # not on a GPU
    ]
    lse = torch.zeros(2, 4, 5)
    bad += [
        (ValueError, lambda: ops.attention_backward(dout[:, :4], q, k, v, q, lse)),
        (TypeError, lambda: ops.attention_backward(dout.float(), q, k, v, q, lse)),
        (ValueError, lambda: ops.attention_backward(dout, q, k, v, q, lse[:, :2])),
        (TypeError, lambda: ops.attention_backward(dout, q, k, v, q, lse.double())),
        (ValueError, lambda: ops.attention_backward(dout, q, k, v, q, lse)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_the_c_entry_refuses():
    """What the Python checks keep out is an error code of the C entry too, before it touches the device."""
    import ctypes
    import train_abi as A
    lib = A.library()
    assert lib.tcpxb_attention_forward(None, None) == -1 and b"null" in lib.tcpxb_train_last_error()

    def args(**kw):
        a = A.Attention(b=1, sq=4, sk=4, heads=4, kv_heads=2, d=64, scale=0.1, dtype=1, out=4096, lse=4096)
        for n in ("q", "k", "v"):
            for field, x in ((n, 4096), (n + "_b", 1024), (n + "_s", 256), (n + "_h", 64)):
                setattr(a, field, x)
        for n, x in kw.items():
            setattr(a, n, x)
        return ctypes.byref(a)

    for kw in ({"b": -1}, {"kv_heads": 3}, {"kv_heads": 0}, {"d": 60}, {"d": 136}, {"d": 0}, {"dtype": 2}, {"scale": 0.0}, {"scale": math.nan},
               {"out": 0}, {"q": 4098}, {"k_s": 257}, {"v": 0}, {"v_s": 0}, {"sk": 1 << 24}):
        assert lib.tcpxb_attention_forward(args(**kw), None) == -1, kw
        assert lib.tcpxb_train_last_error()
    assert lib.tcpxb_attention_backward(args(), None) == -1


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,s,h,hk,d", [(1, 300, 16, 1, 64), (2, 513, 8, 2, 64), (1, 1000, 8, 1, 128), (1, 130, 12, 2, 40), (1, 600, 6, 2, 96)])
def test_shared_tiles_are_summed_over_clusters(b, s, h, hk, d, causal):
    """Few blocks with many tiles each: two, four and eight blocks share a tile; lengths leave some without work."""
    q, k, v, dout = inputs(b, s, s, h, hk, d, BF16, seed=s)
    first = check(q, k, v, dout, causal)
    assert all(torch.equal(x, y) for x, y in zip(first, check(q, k, v, dout, causal)))
    check(q, k, v, dout, causal, torch.full((b,), s // 3, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,sq,sk,h,hk,d", [(1, 1, 4000, 2, 1, 64), (2, 300, 1500, 2, 2, 128), (1, 257, 2100, 1, 1, 64), (1, 20, 3001, 8, 2, 72), (1, 2500, 40, 2, 1, 64)])
def test_long_rows_of_few_queries(b, sq, sk, h, hk, d, dtype):
    """The keys of a row are split over a cluster, whose parts have maxima of their own; some parts are empty."""
    q, k, v, dout = inputs(b, sq, sk, h, hk, d, dtype, seed=sk)
    check(q, k, v, dout)
    check(q, k, v, dout, True)
    lens = torch.tensor([sk // 5, 3][:b], dtype=torch.int32, device="cuda")
    check(q, k, v, dout, False, lens)
    check(q, k, v, dout, True, torch.zeros_like(lens))
    # maxima that rise and fall from part to part
    k[..., 0] = torch.linspace(-20, 20, sk, device="cuda").to(dtype)[None, :, None]
    q[..., 0] = 4.0
    check(q, k, v, dout)
    k[..., 0] = k[..., 0].flip(1)
    check(q, k, v, dout)
    k[:, sk // 2] = math.nan
    assert ops.attention_forward(q, k, v)[0].isnan().all()


def gradients_of(q, k, v, dout, out, lse, causal, lengths=None, scale=None):
    """{name: (value, tolerance)} of dq, dk and dv as functions of what the backward call gets, in 64 bits: the probabilities come
    from the given lse, and D from the given out, or from the row itself where its keys lie in one tile.  Roundings to the type: probabilities, score gradients and results; the rest
    is 32-bit, as in train_oracle.  Under float16's normal range an operand would be off by half of its smallest step, 2^-25.
    Probabilities are lifted by 2^14, score gradients by 2^e with 2^13 <= 2^e X, where X = d max|dout| max|v| over a key head's
    rows that see a key and keys that are seen: that leaves 2^-39 and 2^-38 X."""
    (b, sq, h, d), (sk, hk), u, f32 = q.shape, k.shape[1:3], oracle.half(q.dtype), oracle.F32
    scale = d ** -0.5 if scale is None else scale
    ok = oracle.visible(b, sq, sk, causal, lengths).cuda()
    q, out, dout = (t.double().transpose(1, 2) for t in (q, out, dout))
    seen = ok.expand(b, 1, sq, sk).any(2)[..., None]  # [b, 1, sk, 1]
    k, v = (torch.where(seen, t.double().transpose(1, 2), 0.0).repeat_interleave(h // hk, 1) for t in (k, v))
    p = torch.where(ok, (scale * (q @ k.mT) - lse.double()[..., None]).exp(), 0.0)
    ep = (d + 8) * f32 * scale * (q.abs() @ k.abs().mT) + 8 * f32 * lse.double().abs().nan_to_num(posinf=0.0)[..., None] + 16 * f32
    sees = ok.expand(b, 1, sq, sk).any(-1, keepdim=True)
    x = d * (torch.where(sees, dout, 0.0).abs().amax((2, 3)) * v.abs().amax((2, 3))).unflatten(1, (hk, h // hk)).amax(2).repeat_interleave(h // hk, 1)[..., None, None]
    dp, delta = dout @ v.mT, (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    either = ((p * dp).sum(-1, keepdim=True) - delta).abs()
    eds = ds.abs() * (u + ep) + p * (1 + u) * (either + (d + 8) * f32 * (dout.abs() @ v.abs().mT + (dout * out).abs().sum(-1, keepdim=True)))
    eds, edp = torch.where(ok, eds + x * 2.0 ** -38, 0.0), torch.where(ok, p * (u + ep) + 2.0 ** -39, 0.0)
    n, group = max(sq, sk) + 8, h // hk
    least = torch.finfo(torch.float16).smallest_normal * torch.finfo(torch.float16).eps
    shared = lambda t: t.unflatten(1, (hk, group)).sum(2)  # noqa: E731
    dq, dk, dv = scale * (ds @ k), shared(scale * (ds.mT @ q)), shared(p.mT @ dout)
    edq = u * dq.abs() + scale * ((eds + n * f32 * ds.abs()) @ k.abs())
    edk = u * dk.abs() + shared(scale * ((eds + group * n * f32 * ds.abs()).mT @ q.abs()))
    edv = u * dv.abs() + shared((edp + group * n * f32 * p).mT @ dout.abs())
    return {name: (t.transpose(1, 2), e.transpose(1, 2) * 1.001 + least) for name, t, e in (("dq", dq, edq), ("dk", dk, edk), ("dv", dv, edv))}


def check_gradients(q, k, v, dout, causal=False, lengths=None, scale=None):
    how = {"causal": causal, "key_lengths": lengths, "scale": scale}
    out, lse = ops.attention_forward(q, k, v, **how)
    got = dict(zip(("dq", "dk", "dv"), ops.attention_backward(dout, q, k, v, out, lse, **how)))
    for name, want in gradients_of(q, k, v, dout, out, lse, causal, lengths, scale).items():
        oracle.close(got[name], want, name)
    return got


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("b,sq,sk,h,hk,d", [(1, 2048, 2048, 4, 2, 64), (1, 2048, 2048, 2, 1, 128), (1, 300, 4096, 1, 1, 64), (2, 60, 50, 2, 1, 40), (1, 1500, 1024, 8, 1, 72)])
def test_small_gradients_in_float16(b, sq, sk, h, hk, d, size, causal):
    """Probabilities of thousands of keys times gradients of 1e-3 to 1e-5: score gradients under float16's smallest step."""
    q, k, v, dout = inputs(b, sq, sk, h, hk, d, F16, seed=16)
    check_gradients(q, k, v, (dout.float() * size).half(), causal)


@gpu
def test_probabilities_of_very_many_keys_in_float16():
    """At 2^17 keys a probability is 2^-17, which float16 holds with seven bits."""
    check_gradients(*inputs(1, 64, 1 << 17, 1, 1, 64, F16, seed=17))


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_large_gradients_in_float16(d):
    """Products of dout and v beyond float16's range, whose gradients are within it; peaked and flat rows."""
    for spread in (0.1, 3.0):
        q, k, v, dout = inputs(1, 400, 400, 2, 1, d, F16, seed=18)
        got = check_gradients((q.float() * 30).half(), (k.float() * 30).half(), (v.float() * 100).half(), (dout.float() * 300).half(), True, scale=spread / (900 * d ** 0.5))
        assert all(t.isfinite().all() for t in got.values())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_what_no_row_sees_does_not_take_bits(d, dtype):
    """Large values behind a length, and large gradients of rows that see nothing, leave the others' small ones their bits."""
    q, k, v, dout = inputs(2, 200, 300, 4, 2, d, dtype, seed=19)
    dout = (dout.float() * 1e-5).to(dtype)
    lens = torch.tensor([300, 130], dtype=torch.int32, device="cuda")
    want = check_gradients(q, k, v, dout, False, lens)
    v[1, 130:] = 6e4
    v[1, 200:] = math.nan
    got = check_gradients(q, k, v, dout, False, lens)
    assert all(torch.equal(want[n], got[n]) for n in want)
    q, k, v, dout = inputs(1, 300, 100, 4, 2, d, dtype, seed=20)
    dout = (dout.float() * 1e-5).to(dtype)
    want = check_gradients(q, k, v, dout, True)
    dout[:, :200] = 6e4
    got = check_gradients(q, k, v, dout, True)
    assert all(torch.equal(want[n], got[n]) for n in want)


@gpu
def test_infinite_gradients_in_float16_stay_in_their_heads():
    """A row of infinities (a loss scale that is too large) reaches what it touches and takes no bits from another head's small gradients."""
    q, k, v, dout = inputs(1, 260, 260, 4, 2, 64, F16, seed=21)
    dout = (dout.float() * 1e-5).half()
    want = check_gradients(q, k, v, dout, True)
    dout[:, 77, 0] = math.inf
    out, lse = ops.attention_forward(q, k, v, causal=True)
    got = dict(zip(want, ops.attention_backward(dout, q, k, v, out, lse, causal=True)))
    assert not got["dq"][:, 77, 0].isfinite().any() and not got["dv"][:, 0, 0].isfinite().any()
    got["dq"][:, 77, 0] = want["dq"][:, 77, 0]
    assert torch.equal(got["dq"], want["dq"]) and all(torch.equal(got[n][:, :, 1], want[n][:, :, 1]) for n in want)


@gpu
def test_float16_in_two_graphs():
    """The maxima's scratch is each graph's own: two graphs with gradients of very different sizes replay at the same time."""
    sets = [inputs(2, 260, 700, 4, 2, 64, F16, seed=22 + i) for i in range(2)]
    sets[0][3].mul_(1e-4), sets[1][3].mul_(1e2)
    wanted = []
    for s in sets:
        out, lse = ops.attention_forward(*s[:3])
        wanted.append(ops.attention_backward(s[3], *s[:3], out, lse))
    runs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = ops.attention_forward(*s[:3])
            runs.append((g, ops.attention_backward(s[3], *s[:3], out, lse)))
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, _), st in zip(runs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for want, (_, got) in zip(wanted, runs):
        assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_float16_gradients_need_their_scratch():
    """The C entry refuses float16 gradients without the scratch for their bounds."""
    import ctypes
    import train_abi as A
    lib = A.library()

    class WithBounds(ctypes.Structure):
        _fields_ = [("a", A.Attention), ("bounds", ctypes.c_void_p)]

    a = A.Attention(b=1, sq=4, sk=4, heads=4, kv_heads=2, d=64, scale=0.1, dtype=3, **{n: 4096 for n in "out lse dq dk dv delta".split()})
    for n in ("q", "k", "v", "dout"):
        for field, x in ((n, 4096), (n + "_b", 1024), (n + "_s", 256), (n + "_h", 64)):
            setattr(a, field, x)
    for bounds in (None, 4100):
        assert lib.tcpxb_attention_backward(ctypes.byref(WithBounds(a, bounds)), None) == -1
        assert b"bounds" in lib.tcpxb_train_last_error()
