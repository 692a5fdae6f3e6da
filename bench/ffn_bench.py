#!/usr/bin/env python3
"""Times of the feed-forward operators (csrc/ffn_*.hip) by part: forward, each product of the backward pass, companions, and the two
rates they are priced against (a large copy, a large bf16 library product).

    python bench/ffn_bench.py                        # all
    python bench/ffn_bench.py --only gated           # names that contain the word
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch

from ddl import ops

ap = argparse.ArgumentParser()
ap.add_argument("--only", default="")
ap.add_argument("--iters", type=int, default=20)
a = ap.parse_args()
dev = torch.device("cuda", 0)
ext = ops.require_ext()
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def timeit(fn):
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    s.record()
    for _ in range(a.iters):
        fn()
    e.record()
    torch.cuda.synchronize()
    return s.elapsed_time(e) / a.iters * 1e3


def row(name, fn, flops=0.0, nbytes=0.0):
    if any(w in name for w in a.only.split("|")):
        us = timeit(fn)
        print(f"{name:52s} {us:10.2f} us  {flops / us / 1e6:8.1f} TFLOP/s  {nbytes / us / 1e3:8.1f} GB/s", flush=True)


def rnd(dtype, *shape, scale=1.0):
    return (torch.randn(*shape, device=dev) * scale).to(DT[dtype])


big = torch.empty(2 ** 28, dtype=torch.float32, device=dev)
out = torch.empty_like(big)
row("rate: copy of 1 GiB", lambda: out.copy_(big), nbytes=2.0 * big.numel() * 4)
m, n = rnd("bf16", 8192, 8192), rnd("bf16", 8192, 8192)
row("rate: library product 8192^3 bf16", lambda: m @ n.t(), flops=2.0 * 8192 ** 3)
m, n = rnd("fp32", 4096, 4096), rnd("fp32", 4096, 4096)
row("rate: library product 4096^3 fp32", lambda: m @ n.t(), flops=2.0 * 4096 ** 3)
del big, out, m, n

for dt, M, K, N in (("bf16", 8192, 4096, 4096), ("fp16", 777, 1021, 1531), ("fp32", 30, 1024, 4096), ("fp32", 4096, 4096, 4096),
                    ("bf16", 1, 4096, 4096), ("bf16", 512, 1024, 4096), ("bf16", 64, 4096, 4096)):
    x, w, b, r, dy = rnd(dt, M, K), rnd(dt, N, K, scale=K ** -0.5), rnd(dt, N), rnd(dt, M, N), rnd(dt, M, N)
    f, name, e = 2.0 * M * K * N, f"linear {dt} {M}x{K}x{N}", x.element_size()
    y, z = ext.linear_forward(x, w, b, r, 3, True)
    row(f"{name} forward", lambda: ext.linear_forward(x, w, b, r, 3, False), f, e * (M * K + N * K + 2 * M * N))
    row(f"{name} forward, sums kept", lambda: ext.linear_forward(x, w, b, r, 3, True), f, e * (M * K + N * K + 2 * M * N) + 4 * M * N)
    row(f"{name} dx", lambda: ext.linear_backward(dy, x, w, None, 0, True, False, False), f)
    row(f"{name} dw", lambda: ext.linear_backward(dy, x, w, None, 0, False, True, False), f)
    row(f"{name} db, act'", lambda: ext.linear_backward(dy, x, w, z, 3, False, False, True), 0, (4 + e) * M * N)
for dt, M, K, F in (("bf16", 8192, 4096, 8192), ("bf16", 2011, 1000, 2708), ("fp32", 128, 1024, 4096), ("bf16", 1, 4096, 11264)):
    x, g, u, dy = rnd(dt, M, K), rnd(dt, F, K, scale=K ** -0.5), rnd(dt, F, K, scale=K ** -0.5), rnd(dt, M, F)
    f, name, e = 4.0 * M * K * F, f"gated {dt} {M}x{K}x{F}", x.element_size()
    h, z = ext.gated_forward(x, g, u, None, None, 2, True)
    row(f"{name} forward", lambda: ext.gated_forward(x, g, u, None, None, 2, False), f, e * (M * K + 2 * F * K + M * F))
    row(f"{name} forward, sums kept", lambda: ext.gated_forward(x, g, u, None, None, 2, True), f)
    row(f"{name} dx", lambda: ext.gated_backward(dy, x, g, u, z, 2, True, False, False), f)
    row(f"{name} dw", lambda: ext.gated_backward(dy, x, g, u, z, 2, False, True, False), f)
    row(f"{name} dx, dw", lambda: ext.gated_backward(dy, x, g, u, z, 2, True, True, False), 2 * f)
for dt, M, C in (("bf16", 16384, 8192), ("fp32", 4096, 1024)):
    x, r = rnd(dt, M, C), rnd(dt, M, C)
    key = torch.tensor([1, 2], device=dev)
    row(f"dropout {dt} {M}x{C}", lambda: ext.dropout(x, 0.1, key, None), nbytes=2.0 * x.numel() * x.element_size())
    row(f"dropout {dt} {M}x{C} residual", lambda: ext.dropout(x, 0.1, key, r), nbytes=3.0 * x.numel() * x.element_size())
for dt, M, C in (("bf16", 16384, 4096), ("bf16", 16384, 1024), ("bf16", 8192, 8192), ("fp32", 8192, 2048)):
    x, y, dr, dh = (rnd(dt, M, C) for _ in range(4))
    v = rnd(dt, C)
    args = (x, y, v, v, v, v, v, True, 1e-6, 0.5)
    _, _, st = ext.norm_forward(*args)
    row(f"norm {dt} {M}x{C} forward", lambda: ext.norm_forward(*args), nbytes=4.0 * x.numel() * x.element_size())
    row(f"norm {dt} {M}x{C} backward", lambda: ext.norm_backward(*args, st, dr, dh), nbytes=6.0 * x.numel() * x.element_size())
