"""Feed-forward operators on the CPU (plain PyTorch path): formulas, generator, refusals."""
import pytest
import torch

import ffn_oracle as oracle
from ddl import ops

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rnd(dtype, *shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def same(got, want, dtype, size=1.0):
    """64-bit value against one rounding plus fp32 arithmetic over at most 64 terms of `size`"""
    assert got.dtype == dtype
    off = (got.double() - want).abs()
    assert (off <= oracle.rounding(dtype) * want.abs() + 128 * 2.0 ** -24 * (size + want.abs())).all(), off.max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
def test_products(dtype, act):
    x, w, u = rnd(dtype, 2, 5, 24, seed=1), rnd(dtype, 7, 24, seed=2), rnd(dtype, 7, 24, seed=3)
    b, c, r = rnd(dtype, 7, seed=4), rnd(dtype, 7, seed=5), rnd(dtype, 2, 5, 7, seed=6)
    d = [t.double() for t in (x, w, u, b, c, r)]
    size = (d[0].abs() @ d[1].abs().T).max().item() * (d[0].abs() @ d[2].abs().T).max().item()
    same(ops.linear(x, w, b, activation=act, residual=r), oracle.linear(d[0], d[1], d[3], act, d[5]), dtype, size)
    same(ops.gated_linear(x, w, u, b, c, activation=act), oracle.gated(d[0], d[1], d[2], d[3], d[4], act), dtype, size)
    for t in (x, w, b, r):
        t.requires_grad_(True)
    ops.linear(x, w, b, activation=act, residual=r).sum().backward()
    assert all(t.grad is not None and t.grad.dtype == dtype for t in (x, w, b, r))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
def test_residual_norm(dtype, kind, post, gate):
    x, y = rnd(dtype, 3, 4, 40, seed=1), rnd(dtype, 3, 4, 40, seed=2)
    a = dict(pre_weight=rnd(dtype, 40, seed=3), post_weight=rnd(dtype, 40, seed=4) if post else None,
             gate={"none": None, "channel": rnd(dtype, 40, seed=5), "full": rnd(dtype, 3, 4, 40, seed=5)}[gate])
    if kind == "layer":
        a["pre_bias"] = rnd(dtype, 40, seed=6)
    r, h = ops.residual_norm(x, y, kind=kind, scale=0.5, **a)
    wr, wh = oracle.residual_norm(x.double(), y.double(), kind=kind, scale=0.5, **{k: v.double() if v is not None else None for k, v in a.items()})
    same(r, wr, dtype, 30.0)
    same(h, wh, dtype, 30.0)
    r, h = ops.residual_norm(x, kind=kind, pre_weight=a["pre_weight"])
    assert r is x
    same(h, oracle.norm(x.double(), a["pre_weight"].double(), None, kind, 1e-6), dtype, 30.0)


def test_generator_known_answers():
    """Philox4x32 with 10 and 7 rounds on the zero block, as published with the generator."""
    assert oracle.philox4x32((0,) * 4, (0, 0), 10) == (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)
    assert oracle.philox4x32((0,) * 4, (0, 0), 7) == (0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48)


@pytest.mark.parametrize("n", [0, 1, 5, 64, 1001])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
def test_dropout(n, p):
    for key in [(0, 0), (-5, 2 ** 50 + 3), (2 ** 62, 9)]:
        keep = torch.from_numpy(oracle.kept(key, n, p)).double()
        x, res = rnd(torch.float32, n, seed=1).requires_grad_(True), rnd(torch.float32, n, seed=2)
        y = ops.dropout(x, p, torch.tensor(key), residual=res)
        scale = 1 / (1 - p) if p < 1 else 0.0
        same(y.detach(), x.detach().double() * keep * scale + res.double(), torch.float32, 4.0)
        (dx,) = torch.autograd.grad(y.sum(), x)
        same(dx, keep * scale, torch.float32)
    bad = torch.full((1000,), float("nan"))
    assert (ops.dropout(bad, 1.0, torch.tensor([1, 2])) == 0).all()


def test_dropout_rng():
    rng = ops.DropoutRng(2 ** 63 + 5, "cpu", stream=2)
    assert rng.keys(2).tolist() == [[5 - 2 ** 63, 2 << 48], [5 - 2 ** 63, (2 << 48) + 1]]
    assert rng.next_key().tolist() == [5 - 2 ** 63, (2 << 48) + 2]


def test_refusals():
    x, w, b, n, key = rnd(torch.float32, 4, 8), rnd(torch.float32, 6, 8), rnd(torch.float32, 6), torch.ones(8), torch.tensor([1, 2])
    bad = [
        lambda: ops.linear(x, w[:, :7]), lambda: ops.linear(x, w.bfloat16()), lambda: ops.linear(x, w, b[:5]),
        lambda: ops.linear(x, w, b, residual=x), lambda: ops.linear(x.double(), w.double()), lambda: ops.linear(x, w, activation="tanh"),
        lambda: ops.gated_linear(x, w, w[:5]), lambda: ops.gated_linear(x, w, w, b), lambda: ops.dropout(x, 1.5, key),
        lambda: ops.dropout(x, 0.5, key[:1]), lambda: ops.dropout(x, 0.5, key.float()), lambda: ops.dropout(x, 0.5, key, residual=w),
        lambda: ops.DropoutRng(0, "cpu", stream=-1), lambda: ops.residual_norm(x), lambda: ops.residual_norm(x, gate=n, pre_weight=n),
        lambda: ops.residual_norm(x, x[:3]), lambda: ops.residual_norm(x, pre_weight=n, pre_bias=n),
        lambda: ops.residual_norm(x, x, kind="batch"), lambda: ops.residual_norm(x, x, pre_weight=n[:7]),
        lambda: ops.residual_norm(x, x, pre_weight=n, gate=n.half()), lambda: ops.residual_norm(x, x, gate=x[:2]),
        lambda: ops.residual_norm(x, x, eps=-1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_forward_mode_is_right_or_refused():
    """The plain path has tangents; the kernels have none and refuse a dual tensor, before they look at anything else of it."""
    import torch.autograd.forward_ad as fwd
    x, w, b = rnd(torch.float32, 4, 8, seed=1), rnd(torch.float32, 8, 8, seed=2), rnd(torch.float32, 8, seed=3)
    v, key = torch.ones(8), torch.tensor([1, 2])
    with fwd.dual_level():
        for i in range(3):
            a = [x, w, b]
            t = torch.ones_like(a[i])
            a[i] = fwd.make_dual(a[i], t)
            got = fwd.unpack_dual(ops.linear(*a)).tangent
            want = (lambda: t @ w.T, lambda: x @ t.T, lambda: t.expand(4, 8))[i]()
            same(got, want.double(), torch.float32, 64.0)
        ext = ops.load_ext()
        if ext is None:
            pytest.skip("extension not built")
        d, dw, db = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, b))
        dv = fwd.make_dual(v, v)
        norm = [x, x, v, v, v, v, v]
        calls = [lambda: ext.linear(d, w, b, x, 0), lambda: ext.linear(x, dw, b, x, 0), lambda: ext.linear(x, w, db, x, 0),
                 lambda: ext.linear(x, w, b, d, 0), lambda: ext.linear_forward(d, w, b, x, 0, False),
                 lambda: ext.gated_linear(d, w, w, b, b, 2), lambda: ext.gated_linear(x, dw, w, b, b, 2),
                 lambda: ext.gated_linear(x, w, dw, b, b, 2), lambda: ext.gated_linear(x, w, w, db, b, 2),
                 lambda: ext.gated_linear(x, w, w, b, db, 2), lambda: ext.dropout(d, 0.5, key, None), lambda: ext.dropout(x, 0.5, key, d)]
        for i in range(7):
            args = list(norm)
            args[i] = d if i < 2 else dv
            calls.append(lambda args=args: ext.residual_norm(*args, True, 1e-6, 1.0))
        for i, call in enumerate(calls):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was not refused")


@pytest.mark.filterwarnings("ignore")
def test_recorded_programs_are_right_or_refused():
    """The plain path can be recorded; a kernel's result would be recorded as a constant, so its call refuses, before anything else."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, v, key = rnd(torch.float32, 4, 8, seed=1), rnd(torch.float32, 8, 8, seed=2), torch.ones(8), torch.tensor([1, 2])
    other = rnd(torch.float32, 4, 8, seed=3)
    for record in (lambda f: torch.jit.trace(f, (x,), check_trace=False), lambda f: make_fx(f)(x)):
        plain = record(lambda t: ops.linear(t, w, activation="silu"))
        assert torch.equal(plain(other), ops.linear(other, w, activation="silu"))
        ext = ops.load_ext()
        if ext is None:
            pytest.skip("extension not built")
        for call in (lambda t: ext.linear(t, w, None, None, 0), lambda t: ext.gated_linear(t, w, w, None, None, 2),
                     lambda t: ext.dropout(t, 0.5, key, None), lambda t: ext.rng_keys(key, 1),
                     lambda t: ext.residual_norm(t, None, None, None, None, v, None, False, 1e-6, 1.0)[1]):
            with pytest.raises(NotImplementedError, match="recorded"):
                record(call)


def test_plans_of_the_large_products():
    """tests/test_gpu_ffn_edges.py reaches the large tiles through these sizes: the cost rule still gives them."""
    from test_gpu_ffn_edges import LARGE
    ext = ops.load_ext()
    if ext is None:
        pytest.skip("extension not built")
    for (gated, M, K, N), plans in LARGE.items():
        for name in ("bf16", "fp16"):
            assert [ext.product_plan(what, name, M, K, N, gated) for what in ("forward", "dx", "dw")] == plans, (gated, M, K, N)
    for bad in (("back", "bf16"), ("dx", "int8")):
        with pytest.raises(ValueError):
            ext.product_plan(*bad, 64, 64, 64, False)


def test_channel_gate_beside_a_single_row():
    """A vector may be fp32 beside a 16-bit row, the gate of a single row [C] as well."""
    for dtype in TYPES:
        x, y, g, w = (rnd(t, 40, seed=i) for i, t in enumerate((dtype, dtype, torch.float32, torch.float32)))
        got, want = ops.residual_norm(x, y, gate=g, pre_weight=w), ops.residual_norm(x[None], y[None], gate=g, pre_weight=w)
        assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    with pytest.raises(ValueError):                                  # vectors of two types
        ops.residual_norm(x, y, gate=g, pre_weight=w.to(dtype))


def test_plans_fit_a_launch():
    """A launch has fewer than 2^32 threads: the tiles of many rows are large enough for that (256 threads for 128 x 128, 512 else)."""
    ext = ops.load_ext()
    if ext is None:
        pytest.skip("extension not built")
    for name in ("fp32", "bf16", "fp16"):
        for what, M, K, N, gated in (("forward", 2 ** 28 + 3, 8, 8, False), ("forward", 2 ** 30, 8, 5, False),
                                     ("forward", 2 ** 28, 8, 64, True), ("dx", 2 ** 29, 64, 8, True), ("dw", 2 ** 29, 2 ** 26, 5, False)):
            rows, cols, _ = ext.product_plan(what, name, M, K, N, gated)
            m, n, outs = {"forward": (M, N, 1), "dx": (M, K, 1), "dw": (N, K, 1 + gated)}[what]
            tiles = -(-m // rows) * -(-n // cols) * outs
            assert tiles * (256 if rows == 128 and cols in (64, 128) else 512) < 2 ** 32, (name, what, M, K, N, gated)
    with pytest.raises(ValueError):
        ext.product_plan("forward", "fp32", 64, 2 ** 26 + 1, 64, False)
    with pytest.raises(ValueError):
        ext.product_plan("forward", "fp32", 2 ** 30 + 1, 64, 64, False)


FAR = (1e4, 1e12, 1e20, 1e30)


def check_far_sums(device):
    """Activations and slopes of sums far from zero are their limits, with no infinity or NaN on the way."""
    for act in ops.ACTIVATIONS:
        for z in FAR:
            for sign in (1.0, -1.0):
                x = torch.full((3, 1), sign * z ** 0.5, device=device, requires_grad=True)
                w = torch.full((1, 1), z ** 0.5, device=device, requires_grad=True)
                value = {"none": sign * z, "sigmoid": max(sign, 0.0)}.get(act, max(sign, 0.0) * z)
                slope = {"none": 1.0, "sigmoid": 0.0}.get(act, max(sign, 0.0))
                y = ops.linear(x, w, activation=act)
                dx, dw = torch.autograd.grad(y.sum(), (x, w))
                for got, want in ((y, value), (dx, slope * z ** 0.5), (dw, 3 * slope * sign * z ** 0.5)):
                    torch.testing.assert_close(got, torch.full_like(got, want), rtol=1e-5, atol=1e-30)
                up = (w.detach() / z).requires_grad_(True)             # x times this: the sign
                h = ops.gated_linear(x, w, up, activation=act)
                torch.testing.assert_close(h, torch.full_like(h, value * sign), rtol=1e-5, atol=1e-30)
                (dw,) = torch.autograd.grad(h.sum(), w)
                torch.testing.assert_close(dw, torch.full_like(dw, 3 * slope * z ** 0.5), rtol=1e-5, atol=1e-30)


def test_far_sums():
    check_far_sums("cpu")
