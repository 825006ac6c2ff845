"""One small, fixed workload per kernel of this library, for profiler captures.

    python -m nccl_plugin_gpudirecttcpx_b200.ops.profile_case --kernel reduce_fanout
    ncu --set full --clock-control none -k regex:unpack_kernel -s 2 -c 1 -o prof \
        python -m nccl_plugin_gpudirecttcpx_b200.ops.profile_case --kernel reduce_fanout

Every case moves 64 MiB assembled from 16 384 fragments of 4096 bytes at permuted offsets of
a 256 MiB pool (larger than L2, well under a GB on the device in total), bf16 payload, and
launches its kernel `--iters` times (default 3) after nothing else: a capture of launch 3
(`-s 2 -c 1`) sees a warmed-up kernel and ends in seconds.  One GPU: the "peers" of the fan-out
kernels are three more buffers on the same device, so the capture shows the kernel's
instruction mix and memory traffic, not NVLink.  Prints one JSON line with the CUDA-event time
of the last launch.

The training operators' cases: attention and its backward pass over 2 x 2048 tokens, 32/8 heads of 64
(`--head-size 128`: 4096 tokens, 16/4 heads), causal, bf16; head norms with rotation of 4 x 2048 tokens,
32/8 heads of 64; AdamW over 128 M bf16 weights with states in 32 or 8 bits.
"""
from __future__ import annotations

import argparse
import json
import sys

TRAINING = ("attention", "attention_backward", "norm_rope", "norm_rope_backward", "adamw", "adamw_8bit")
KERNELS = ("copy", "reduce", "reduce_l2", "fanout", "reduce_fanout", "peer_reduce", "checksum", "copy_host_pool", "reduce_host_pool", *TRAINING)


def training_case(kernel: str, head_size: int):
    """A call of one training operator on inputs of its own."""
    import torch
    from .. import ops

    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)

    if kernel.startswith("attention"):
        b, s, h, hk = (2, 2048, 32, 8) if head_size <= 64 else (1, 4096, 16, 4)
        q, k, v, dout = normal(b, s, h, head_size), normal(b, s, hk, head_size), normal(b, s, hk, head_size), normal(b, s, h, head_size)
        if kernel == "attention":
            return lambda: ops.attention_forward(q, k, v, causal=True)
        out, lse = ops.attention_forward(q, k, v, causal=True)
        return lambda: ops.attention_backward(dout, q, k, v, out, lse, causal=True)
    if kernel.startswith("norm_rope"):
        q, k = normal(4, 2048, 32, 64), normal(4, 2048, 8, 64)
        angle = torch.outer(torch.arange(2048, device="cuda"), 5e5 ** (-torch.arange(0, 64, 2, device="cuda") / 64))
        args = angle.cos(), angle.sin(), normal(64), normal(64)
        dq, dk = normal(*q.shape), normal(*k.shape)
        if kernel == "norm_rope":
            return lambda: ops.qk_norm_rope(q, k, *args)
        return lambda: ops.qk_norm_rope_backward(dq, dk, q, k, *args)
    n = 128 << 20
    kind = torch.float32 if kernel == "adamw" else torch.float8_e4m3fn
    m, v = (torch.zeros(n, dtype=kind, device="cuda") for _ in range(2))
    scales = {} if kernel == "adamw" else {name: [torch.zeros(n // 256, device="cuda")] for name in ("exp_avg_scales", "exp_avg_sq_scales")}
    p, grad, steps = normal(n), normal(n), torch.zeros(1, dtype=torch.int32, device="cuda")
    return lambda: ops.adamw_step([p], [grad], [m], [v], steps, lr=1e-4, **scales)


def timed(call, iters: int) -> float:
    """Milliseconds of the last of `iters` calls."""
    import torch
    ms = 0.0
    for _ in range(max(iters, 1)):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        call()
        e1.record()
        torch.cuda.synchronize()
        ms = e0.elapsed_time(e1)
    return ms


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--kernel", choices=KERNELS, required=True)
    ap.add_argument("--iters", type=int, default=3)
    ap.add_argument("--mb", type=int, default=64, help="bytes assembled per launch (MiB)")
    ap.add_argument("--ctas", type=int, default=0, help="CTA limit of the unpack kernels (0 = one per SM)")
    ap.add_argument("--head-size", type=int, default=64, help="of the attention cases")
    args = ap.parse_args(argv)

    import torch
    from . import unpack as U
    from .. import ops

    if args.kernel in TRAINING:
        call = training_case(args.kernel, args.head_size)
        print(json.dumps({"kernel": args.kernel, "iters": args.iters, "last_launch_us": round(timed(call, args.iters) * 1e3, 2)}))
        return 0
    dev = torch.device("cuda")
    total = args.mb << 20
    pool_bytes = 256 << 20
    g = torch.Generator(device=dev).manual_seed(1)
    pool = torch.randn(pool_bytes // 2, device=dev, generator=g).to(torch.bfloat16)
    if args.kernel in ("copy_host_pool", "reduce_host_pool"):
        # the transport's default rx pool placement: pinned host memory the kernel reads over PCIe
        host = torch.empty(pool_bytes // 2, dtype=torch.bfloat16).pin_memory()
        host.copy_(pool)
        pool = host
    descs = U.descriptors_to_device(U.permuted_fragments(total, pool_bytes, seed=5))
    n_el = total // 2
    dst = torch.randn(n_el, device=dev, generator=g).to(torch.bfloat16)
    peers = [torch.empty(n_el, dtype=torch.bfloat16, device=dev) for _ in range(3)]
    st = U.status_buffer()
    flat = torch.randn(total // 2, device=dev, generator=g).to(torch.bfloat16)
    srcs = [flat] + peers
    out_q = torch.empty(n_el // 4, dtype=torch.bfloat16, device=dev)
    kw = {"max_ctas": args.ctas} if args.ctas else {}

    def run():
        k = args.kernel
        if k in ("copy", "copy_host_pool"):
            U.unpack_copy(pool, dst, descs, status=st, **kw)
        elif k in ("reduce", "reduce_host_pool"):
            U.unpack_reduce(pool, dst, descs, status=st, **kw)
        elif k == "reduce_l2":
            U.unpack_reduce(pool, dst, descs, status=st, impl=U.REDUCE_L2, **kw)
        elif k == "fanout":
            U.unpack_fanout(pool, dst, peers, descs, status=st, **kw)
        elif k == "reduce_fanout":
            U.unpack_reduce_fanout(pool, dst, dst, peers, descs, status=st, **kw)
        elif k == "peer_reduce":
            # the intra-node reduce-scatter stage: a quarter of four 64 MiB buffers summed
            ops.peer_reduce(out_q, srcs, shard_off=(total // 4))
        elif k == "checksum":
            ops.checksum(flat.view(torch.uint8))

    ms = timed(run, args.iters)
    print(json.dumps({"kernel": args.kernel, "mb": args.mb, "iters": args.iters, "last_launch_us": round(ms * 1e3, 2),
                      "status": st.tolist()[0]}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
