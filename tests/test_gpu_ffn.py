"""Feed-forward operators on the GPU against their formulas in 64 bits (tests/ffn_oracle.py).

Tolerances are element-wise bounds, written down before the first run.  EPS = 2^-24 is the rounding of fp32, u that of the
output's type (half a step).  A sum of n products in fp32 is off by at most (n + 16) EPS times the sum of their absolute values,
whatever its order; an activation has slope <= 1.13 and its derivative slope <= 1.2 (silu, gelu), each evaluated to 16 EPS.
"""
import pytest
import torch

import ffn_oracle as oracle

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from ddl import ops
    ops.require_ext()
    return torch.device("cuda", 0)


def rnd(dev, dtype, *shape, seed=0, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + sum(shape) + len(shape))
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def tiny(dtype):
    """half the smallest step of fp16 (bf16 and fp32 reach far below any value here)"""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def close(got, want, bound, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, (what, got.dtype, got.shape, want.shape)
    if want.numel() == 0:
        return
    limit = oracle.rounding(dtype) * (want.abs() + bound) + bound + tiny(dtype)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off / limit).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound, largest difference {off.max().item():.3e}"


def product_bounds(x, w, b, act):
    """(z, bound of z) in 64 bits"""
    z = x @ w.T
    mag = x.abs() @ w.abs().T
    if b is not None:
        z, mag = z + b, mag + b.abs()
    return z, (x.shape[1] + 16) * EPS * mag


def act_and_slope(z, act):
    zz = z.clone().requires_grad_(True)
    a = oracle.ACTS[act](zz)
    (da,) = torch.autograd.grad(a.sum(), zz)
    return a.detach(), da


def slope_bound(z, zerr, act):
    """how far act'(z) may be off: relu jumps where z may have the other sign"""
    if act == "none":
        return torch.zeros_like(z)
    if act == "relu":
        return (z.abs() <= zerr).double()
    return 1.2 * zerr + 16 * EPS * (1 + z.abs())


def check_linear(dev, dtype, x, w, b, act, res, backward=True):
    from ddl import ops
    leaves = [t.requires_grad_(True) if t is not None else None for t in (x, w, b, res)]
    y = ops.linear(x, w, b, activation=act, residual=res)
    X, W, B, R = [t.detach().double() if t is not None else None for t in leaves]
    X2 = X.reshape(X.shape[:-1].numel(), X.shape[-1])
    z, zerr = product_bounds(X2, W, B, act)
    a, da = act_and_slope(z, act)
    want, bound = a, 1.13 * zerr + (16 * EPS * (a.abs() + z.abs()) if act != "none" else 0)
    if R is not None:
        want = want + R.reshape(want.shape)
        bound = bound + 2 * EPS * want.abs()
    close(y.reshape(want.shape), want, bound, dtype, "y")
    if not backward:
        return
    dy = rnd(dev, dtype, *y.shape, seed=9)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    got = dict(zip([n for n, t in zip("xwbr", leaves) if t is not None], grads))
    D = dy.double().reshape(want.shape)
    dz = D * da
    e32 = D.abs() * slope_bound(z, zerr, act) + 4 * EPS * dz.abs()
    u = oracle.rounding(dtype) if act != "none" else 0.0
    edz = e32 + u * (dz.abs() + e32) + tiny(dtype)                     # dz is rounded once before its products
    M, N = dz.shape
    close(got["x"].reshape(X2.shape), dz @ W, edz @ W.abs() + (N + 16) * EPS * (dz.abs() @ W.abs()), dtype, "dx")
    close(got["w"], dz.T @ X2, edz.T @ X2.abs() + (M + 16) * EPS * (dz.abs().T @ X2.abs()), dtype, "dw")
    if b is not None:
        close(got["b"], dz.sum(0), e32.sum(0) + (M + 16) * EPS * dz.abs().sum(0), dtype, "db")
    if res is not None:
        assert torch.equal(got["r"], dy)


SHAPES = [(1, 1, 1), (1, 7, 5), (1, 1024, 5), (2, 64, 64), (16, 96, 17), (17, 513, 40), (32, 1000, 31), (33, 65, 129), (40, 4096, 48),
          (64, 128, 256), (127, 63, 130), (129, 256, 257), (300, 520, 140), (1000, 72, 24)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(dev, dtype, M, K, N):
    i = SHAPES.index((M, K, N))
    act = list(oracle.ACTS)[i % 6]
    b = rnd(dev, dtype, N, seed=3) if i % 2 else None
    res = rnd(dev, dtype, M, N, seed=4) if i % 3 else None
    check_linear(dev, dtype, rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5), b, act, res)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", list(oracle.ACTS))
def test_linear_activations(dev, dtype, act):
    x, w = rnd(dev, dtype, 70, 96, seed=1, scale=2.0), rnd(dev, dtype, 50, 96, seed=2, scale=0.3)
    check_linear(dev, dtype, x, w, rnd(dev, dtype, 50, seed=3), act, rnd(dev, dtype, 70, 50, seed=4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=IDS[1:])
@pytest.mark.parametrize("M,K,N", [(4096, 128, 4096), (4000, 200, 3976)])
def test_linear_large_tiles(dev, dtype, M, K, N):
    check_linear(dev, dtype, rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5), rnd(dev, dtype, N, seed=3),
                 "gelu", rnd(dev, dtype, M, N, seed=4))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(0, 8, 5), (4, 0, 6), (40, 0, 6), (4, 8, 0), (0, 0, 0)])
def test_empty_products(dev, dtype, M, K, N):
    """No rows, nothing to sum, no columns: empty results, act(bias) + residual, zero gradients."""
    check_linear(dev, dtype, rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, N, K, seed=2), rnd(dev, dtype, N, seed=3), "gelu",
                 rnd(dev, dtype, M, N, seed=4))
    from ddl import ops
    x, wg, wu = (t.requires_grad_(True) for t in (rnd(dev, dtype, M, K), rnd(dev, dtype, N, K), rnd(dev, dtype, N, K, seed=5)))
    h = ops.gated_linear(x, wg, wu)
    assert h.shape == (M, N) and (h == 0).all()
    for t, g in zip((x, wg, wu), torch.autograd.grad(h.sum(), (x, wg, wu))):
        assert g.shape == t.shape and (g == 0).all()


def layouts(dev, dtype, rows, cols, seed):
    """The same kind of matrix in the layouts a program may hold it in."""
    wide = rnd(dev, dtype, rows, 2 * cols + 3, seed=seed)
    yield "transposed", rnd(dev, dtype, cols, rows, seed=seed).t()
    yield "every other column", wide[:, 1:1 + 2 * cols:2]
    yield "slice off 16 bytes", wide[:, 1:1 + cols]
    yield "slice", rnd(dev, dtype, rows, cols + 64, seed=seed)[:, 32:32 + cols]
    yield "one row repeated", rnd(dev, dtype, 1, cols, seed=seed).expand(rows, cols)
    yield "flipped rows", rnd(dev, dtype, rows, cols, seed=seed).flip(0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [5, 200])
def test_linear_layouts(dev, dtype, M):
    K, N = 72, 48
    base = dict(x=rnd(dev, dtype, M, K, seed=1), w=rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5), res=rnd(dev, dtype, M, N, seed=4))
    for name, rows, cols in (("x", M, K), ("w", N, K), ("res", M, N)):
        for what, t in layouts(dev, dtype, rows, cols, 7):
            a = {k: v.clone() for k, v in base.items()}
            a[name] = t.detach()
            try:
                check_linear(dev, dtype, a["x"], a["w"], None, "silu", a["res"])
            except AssertionError as e:
                raise AssertionError(f"{name} {what}: {e}")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_more_dimensions_and_one_vector(dev, dtype):
    w, b = rnd(dev, dtype, 24, 40, seed=2, scale=0.2), rnd(dev, dtype, 24, seed=3)
    check_linear(dev, dtype, rnd(dev, dtype, 3, 7, 40, seed=1), w, b, "silu", rnd(dev, dtype, 3, 7, 24, seed=4))
    check_linear(dev, dtype, rnd(dev, dtype, 40, seed=1), w, b, "none", rnd(dev, dtype, 24, seed=4))
    check_linear(dev, dtype, rnd(dev, dtype, 5, 9, 40, seed=1).transpose(0, 1), w, b, "relu", None)


def in_nans(dev, t):
    """The tensor as a slice in a field of NaN: whatever is read beside it shows."""
    field = torch.full((t.shape[0] + 8, t.shape[1] + 64), float("nan"), dtype=t.dtype, device=dev)
    v = field[3:3 + t.shape[0], 32:32 + t.shape[1]]
    v.copy_(t)
    return v


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(3, 40, 24), (70, 40, 24), (150, 104, 136), (70, 41, 23)])
def test_nothing_beside_the_operands_enters(dev, dtype, M, K, N):
    x, w = in_nans(dev, rnd(dev, dtype, M, K, seed=1)), in_nans(dev, rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5))
    check_linear(dev, dtype, x, w, rnd(dev, dtype, N, seed=3), "gelu", in_nans(dev, rnd(dev, dtype, M, N, seed=4)))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_infinities_stay_in_their_row(dev, dtype):
    from ddl import ops
    for M in (20, 100):
        x, w = rnd(dev, dtype, M, 200, seed=1), rnd(dev, dtype, 70, 200, seed=2)
        want = ops.linear(x, w)
        bad = x.clone()
        bad[7, 3], bad[11, 5] = float("inf"), float("nan")
        got = ops.linear(bad, w)
        rows = torch.tensor([i for i in range(M) if i not in (7, 11)], device=dev)
        assert torch.equal(got[rows], want[rows])
        assert torch.equal(got[7].isinf(), w[:, 3] != 0) and got[11].isnan().all()
        assert torch.equal(ops.linear(x, w, activation="relu"), want.clamp(min=0))
        assert ops.linear(bad, w, activation="relu")[11].isnan().all()


def check_gated(dev, dtype, x, wg, wu, bg, bu, act):
    from ddl import ops
    leaves = [t.requires_grad_(True) if t is not None else None for t in (x, wg, wu, bg, bu)]
    h = ops.gated_linear(x, wg, wu, bg, bu, activation=act)
    X, G, U, BG, BU = [t.detach().double() if t is not None else None for t in leaves]
    X2 = X.reshape(X.shape[:-1].numel(), X.shape[-1])
    g, gerr = product_bounds(X2, G, BG, act)
    up, uerr = product_bounds(X2, U, BU, act)
    a, da = act_and_slope(g, act)
    aerr = 1.13 * gerr + 16 * EPS * (a.abs() + g.abs())
    want = a * up
    close(h.reshape(want.shape), want, aerr * (up.abs() + uerr) + a.abs() * uerr + 2 * EPS * want.abs(), dtype, "h")
    dy = rnd(dev, dtype, *h.shape, seed=9)
    got = dict(zip([n for n, t in zip(("x", "g", "u", "bg", "bu"), leaves) if t is not None],
                   torch.autograd.grad(h, [t for t in leaves if t is not None], dy)))
    D = dy.double().reshape(want.shape)
    u = oracle.rounding(dtype)
    dg, du = D * up * da, D * a
    serr = slope_bound(g, gerr, act)
    eg = D.abs() * (serr * (up.abs() + uerr) + da.abs() * uerr) + 8 * EPS * dg.abs()
    eu = D.abs() * aerr + 8 * EPS * du.abs()
    M, F = dg.shape
    rg, ru = eg + u * (dg.abs() + eg) + tiny(dtype), eu + u * (du.abs() + eu) + tiny(dtype)
    close(got["x"].reshape(X2.shape), dg @ G + du @ U,
          rg @ G.abs() + ru @ U.abs() + (2 * F + 16) * EPS * (dg.abs() @ G.abs() + du.abs() @ U.abs()), dtype, "dx")
    close(got["g"], dg.T @ X2, rg.T @ X2.abs() + (M + 16) * EPS * (dg.abs().T @ X2.abs()), dtype, "dw_gate")
    close(got["u"], du.T @ X2, ru.T @ X2.abs() + (M + 16) * EPS * (du.abs().T @ X2.abs()), dtype, "dw_up")
    if bg is not None:
        close(got["bg"], dg.sum(0), eg.sum(0) + (M + 16) * EPS * dg.abs().sum(0), dtype, "db_gate")
        close(got["bu"], du.sum(0), eu.sum(0) + (M + 16) * EPS * du.abs().sum(0), dtype, "db_up")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,K,F", [(1, 1, 1), (1, 1024, 300), (15, 130, 47), (32, 64, 64), (33, 100, 129), (130, 72, 200), (40, 4100, 24),
                                   (257, 333, 131)])
def test_gated_linear(dev, dtype, M, K, F):
    act = ["silu", "gelu", "gelu_tanh", "sigmoid", "relu", "none"][(M + K) % 6]
    bias = F % 2 == 1
    check_gated(dev, dtype, rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, F, K, seed=2, scale=K ** -0.5),
                rnd(dev, dtype, F, K, seed=3, scale=K ** -0.5), rnd(dev, dtype, F, seed=4) if bias else None,
                rnd(dev, dtype, F, seed=5) if bias else None, act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=IDS[1:])
def test_gated_large_tiles(dev, dtype):
    check_gated(dev, dtype, rnd(dev, dtype, 4096, 136, seed=1), rnd(dev, dtype, 2056, 136, seed=2, scale=0.1),
                rnd(dev, dtype, 2056, 136, seed=3, scale=0.1), None, None, "silu")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [4, 90])
def test_gated_layouts(dev, dtype, M):
    K, F = 56, 40
    base = dict(x=rnd(dev, dtype, M, K, seed=1), g=rnd(dev, dtype, F, K, seed=2, scale=0.2), u=rnd(dev, dtype, F, K, seed=3, scale=0.2))
    for name, rows in (("x", M), ("g", F), ("u", F)):
        for what, t in layouts(dev, dtype, rows, K, 7):
            a = {k: v.clone() for k, v in base.items()}
            a[name] = t.detach()
            try:
                check_gated(dev, dtype, a["x"], a["g"], a["u"], None, None, "gelu")
            except AssertionError as e:
                raise AssertionError(f"{name} {what}: {e}")


# ---- dropout ----------------------------------------------------------------------------------------------------------------
KEYS = [(0, 0), (2 ** 62 + 12345, 3), (-1, (5 << 48) + 7)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n", [0, 1, 3, 4, 7, 8, 9, 1023, 4100])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(dev, dtype, n, p):
    from ddl import ops
    for key in KEYS:
        k = torch.tensor(key, device=dev)
        keep = torch.from_numpy(oracle.kept(key, n, p)).to(dev).double()
        x, res, dy = (rnd(dev, dtype, n, seed=s) for s in (1, 2, 3))
        scale = 1 / (1 - p) if p < 1 else 0.0
        for r in (None, res):
            xg = x.clone().requires_grad_(True)
            rg = r.clone().requires_grad_(True) if r is not None else None
            y = ops.dropout(xg, p, k, residual=rg)
            want = x.double() * keep * scale
            close(y, want if r is None else want + r.double(), 3 * EPS * (want.abs() + (0 if r is None else r.double().abs())), dtype, "y")
            got = torch.autograd.grad(y, [t for t in (xg, rg) if t is not None], dy)
            wdx = dy.double() * keep * scale
            close(got[0], wdx, 2 * EPS * wdx.abs(), dtype, "dx")
            if r is not None:
                assert torch.equal(got[1], dy)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_dropout_does_not_depend_on_layout_and_hides_what_it_drops(dev, dtype):
    from ddl import ops
    k = torch.tensor(KEYS[1], device=dev)
    x = rnd(dev, dtype, 37, 53)
    want = ops.dropout(x, 0.4, k)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.4, k), want)
    odd = torch.empty(37 * 53 + 1, dtype=dtype, device=dev)[1:].view(37, 53)            # not 16-byte aligned
    odd.copy_(x)
    assert torch.equal(ops.dropout(odd, 0.4, k), want)
    dropped = torch.from_numpy(~oracle.kept(KEYS[1], x.numel(), 0.4)).to(dev).view(37, 53)
    bad = torch.where(dropped, torch.full_like(x, float("nan")), x)
    assert torch.equal(ops.dropout(bad, 0.4, k), want)
    assert 0.3 < dropped.double().mean().item() < 0.5


def test_dropout_past_32_bits(dev):
    """Elements beyond 2^31: the last ones of 2^31 + 37 agree with the generator."""
    from ddl import ops
    n = 2 ** 31 + 37
    x = torch.ones(n, dtype=torch.float16, device=dev)
    y = ops.dropout(x, 0.5, torch.tensor(KEYS[1], device=dev))
    seed, call = (int(v) & (2 ** 64 - 1) for v in KEYS[1])
    for first in (0, 2 ** 30, 2 ** 31 - 8, 2 ** 31 + 32):
        words = oracle.philox4x32((first // 4, 0, call & 0xFFFFFFFF, call >> 32), (seed & 0xFFFFFFFF, seed >> 32), 7)
        assert y[first:first + 4].tolist() == [2.0 if w >= 2 ** 31 else 0.0 for w in words]


def test_dropout_rng(dev):
    from ddl import ops
    a, b = ops.DropoutRng(7, dev), ops.DropoutRng(7, dev, stream=3)
    assert a.keys(3).tolist() == [[7, 0], [7, 1], [7, 2]] and a.next_key().tolist() == [7, 3]
    assert b.next_key().tolist() == [7, 3 << 48] and b.next_key().tolist() == [7, (3 << 48) + 1]
    assert ops.DropoutRng(2 ** 64 - 1, dev).next_key().tolist() == [-1, 0]
    assert a.keys(1000).tolist() == [[7, 4 + i] for i in range(1000)]
    c = ops.DropoutRng(7, dev)                                       # a captured take gives new keys on every replay
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        k = c.next_key()
    for i in range(4):
        g.replay()
        assert k.tolist() == [7, 2 * i]
        assert c.next_key().tolist() == [7, 2 * i + 1]               # eager work between the replays


# ---- residual_norm ------------------------------------------------------------------------------------------------------------
DEPTH = 40        # additions on one path of a row sum: 16 a lane, 6 in the wave, up to 16 waves


def hat_bound(v, verr, kind, eps):
    """(hat, rstd, bound of hat, relative bound of rstd) of a norm whose input is off by at most verr"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    c = v - mean
    rstd = 1 / (c.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    hat = c * rstd
    ce = 2 * verr.amax(-1, keepdim=True) + (DEPTH + 2) * EPS * v.abs().mean(-1, keepdim=True) if kind == "layer" \
        else verr.amax(-1, keepdim=True)
    rel = ce * rstd + 2 * DEPTH * EPS
    return hat, rstd, hat.abs() * (rel + 4 * EPS) + ce * rstd, rel


def back_bound(d, derr, hat, herr, rstd, rel, kind):
    """(value, bound) of rstd (d - mean(d) - hat mean(d hat))"""
    m = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    md = m(d) if kind == "layer" else 0.0
    value = rstd * (d - md - hat * m(d * hat))
    size = rstd * (d.abs() + m(d.abs()) + hat.abs() * m((d * hat).abs()))
    bound = size * (rel + 3 * DEPTH * EPS) + rstd * (derr + m(derr) + hat.abs() * m(derr * hat.abs() + d.abs() * herr)
                                                     + herr * m((d * hat).abs()))
    return value, bound


def check_norm(dev, dtype, shape, kind, post, pre, gate, bias, scale=1.0, ptype=None, layout=lambda t: t, eps=1e-6):
    from ddl import ops
    C = shape[-1]
    ptype = ptype or dtype
    t = dict(x=layout(rnd(dev, dtype, *shape, seed=1)), branch=None, gate=None, post_w=None, post_b=None, pre_w=None, pre_b=None)
    if post is not None:
        t["branch"] = layout((rnd(dev, dtype, *shape, seed=2).float() * 2 + 0.5).to(dtype))
        if gate == "channel":
            t["gate"] = rnd(dev, ptype, C, seed=3)
        elif gate == "full":
            t["gate"] = layout(rnd(dev, dtype, *shape, seed=3))
    for name, on in (("post", bool(post)), ("pre", pre)):
        if on:
            t[name + "_w"] = (1 + 0.3 * rnd(dev, torch.float32, C, seed=4)).to(ptype)
            if bias and kind == "layer":
                t[name + "_b"] = rnd(dev, ptype, C, seed=5)
    for v in t.values():
        if v is not None:
            v.requires_grad_(True)
    r, h = ops.residual_norm(t["x"], t["branch"], kind=kind, eps=eps, pre_weight=t["pre_w"], pre_bias=t["pre_b"], post_weight=t["post_w"],
                             post_bias=t["post_b"], gate=t["gate"], scale=scale)
    T = {k: v.detach().double() if v is not None else None for k, v in t.items()}
    zero = torch.zeros_like(T["x"])
    # forward
    want_r, rerr = T["x"], zero
    if post is not None:
        n, nerr = T["branch"], zero
        if post:
            nhat, nrstd, nherr, nrel = hat_bound(T["branch"], zero, kind, eps)
            b = 0 if T["post_b"] is None else T["post_b"]
            n = nhat * T["post_w"] + b
            nerr = nherr * T["post_w"].abs() + 2 * EPS * ((nhat * T["post_w"]).abs() + n.abs())
        g = scale * (1.0 if T["gate"] is None else T["gate"])
        gabs = abs(scale) if T["gate"] is None else g.abs()
        want_r = T["x"] + g * n
        rerr = gabs * nerr + 4 * EPS * (T["x"].abs() + (g * n).abs())
        close(r, want_r, rerr, dtype, "r")
    else:
        assert r is t["x"]
    if pre:
        hat, rstd, herr, rel = hat_bound(want_r, rerr, kind, eps)
        want_h = hat * T["pre_w"] + (0 if T["pre_b"] is None else T["pre_b"])
        close(h, want_h, herr * T["pre_w"].abs() + 4 * EPS * ((hat * T["pre_w"]).abs() + want_h.abs()), dtype, "h")
    else:
        assert h is None
    # backward
    dr = rnd(dev, dtype, *shape, seed=7) if post is not None else None
    dh = rnd(dev, dtype, *shape, seed=8) if pre else None
    outs = [o for o, d in ((r, dr), (h, dh)) if d is not None]
    names = [k for k, v in t.items() if v is not None]
    got = dict(zip(names, torch.autograd.grad(outs, [t[k] for k in names], [d for d in (dr, dh) if d is not None])))
    rows = T["x"].numel() // C
    acc = (rows + 64) * EPS

    def colsum(v, verr):
        return v.reshape(-1, C).sum(0), verr.reshape(-1, C).sum(0) + acc * v.abs().reshape(-1, C).sum(0)

    D, derr = (dr.double(), zero) if dr is not None else (zero, zero)
    if pre:
        DH = dh.double()
        close(got["pre_w"], *colsum(DH * hat, DH.abs() * herr), ptype, "dpre_w")
        if T["pre_b"] is not None:
            close(got["pre_b"], *colsum(DH, zero), ptype, "dpre_b")
        d = DH * T["pre_w"]
        v, e = back_bound(d, 2 * EPS * d.abs(), hat, herr, rstd, rel, kind)
        D, derr = D + v, e + 2 * EPS * (D.abs() + v.abs())
    close(got["x"], D, derr, dtype, "dx")
    if post is None:
        return
    if T["gate"] is not None:
        v, e = scale * n * D, abs(scale) * (n.abs() * derr + nerr * (D.abs() + derr)) + 4 * EPS * (scale * n * D).abs()
        if gate == "channel":
            close(got["gate"], *colsum(v, e), ptype, "dgate")
        else:
            close(got["gate"], v, e, dtype, "dgate")
    dn, dnerr = g * D, gabs * derr + 4 * EPS * (g * D).abs()
    if post:
        close(got["post_w"], *colsum(dn * nhat, dnerr * nhat.abs() + dn.abs() * nherr), ptype, "dpost_w")
        if T["post_b"] is not None:
            close(got["post_b"], *colsum(dn, dnerr), ptype, "dpost_b")
        d = dn * T["post_w"]
        v, e = back_bound(d, (dnerr + 2 * EPS * dn.abs()) * T["post_w"].abs(), nhat, nherr, nrstd, nrel, kind)
        close(got["branch"], v, e, dtype, "dbranch")
    else:
        close(got["branch"], dn, dnerr, dtype, "dbranch")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 4096), (3, 7), (5, 512), (6, 516), (257, 1024), (9, 1030), (33, 2048), (700, 24), (7, 4104),
                                    (3, 8192), (2, 8200), (2, 16384), (5, 16001)])
def test_residual_norm(dev, dtype, kind, rows, C):
    if C == 1 and kind == "layer":
        pytest.skip("a layer norm over one column divides its rounding error by sqrt(eps): no digit of it is defined")
    check_norm(dev, dtype, (rows, C), kind, True, True, "channel", True, scale=0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False), (None, True)])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
def test_residual_norm_forms(dev, dtype, post, pre, gate):
    for kind in ("rms", "layer"):
        for C in (96, 101):
            check_norm(dev, dtype, (13, C), kind, post, pre, gate, bias=C == 96, scale=-1.5)
            if dtype != torch.float32:
                check_norm(dev, dtype, (13, C), kind, post, pre, gate, bias=C == 96, ptype=torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_layouts(dev, dtype):
    check_norm(dev, dtype, (3, 5, 64), "layer", True, True, "full", True)
    check_norm(dev, dtype, (64,), "rms", True, True, "full", False)
    check_norm(dev, dtype, (6, 64), "rms", True, True, "channel", False, layout=lambda t: t.t().contiguous().t().detach())
    check_norm(dev, dtype, (6, 64), "layer", True, True, "full", True,
               layout=lambda t: torch.cat([t, t], 1)[:, 64:].detach())
    check_norm(dev, dtype, (6, 64), "layer", True, True, "full", True,
               layout=lambda t: torch.cat([t.reshape(-1), t.reshape(-1)])[1:385].view(6, 64).detach())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_without_rows_and_far_from_zero(dev, dtype):
    from ddl import ops
    x = torch.empty(0, 48, dtype=dtype, device=dev, requires_grad=True)
    w = torch.ones(48, dtype=dtype, device=dev, requires_grad=True)
    r, h = ops.residual_norm(x, x, pre_weight=w, gate=w)
    assert r.shape == h.shape == (0, 48)
    dx, dw = torch.autograd.grad((r, h), (x, w), (r, h))
    assert dx.shape == (0, 48) and (dw == 0).all()
    # the variance is taken about the mean: rows around 100 with spread 1
    v = (rnd(dev, torch.float32, 5, 1000) + 100).to(dtype)
    one = torch.ones(1000, dtype=dtype, device=dev)
    _, h = ops.residual_norm(v, kind="layer", pre_weight=one)
    hat, _, herr, _ = hat_bound(v.double(), torch.zeros_like(v.double()), "layer", 1e-6)
    close(h, hat, herr + 4 * EPS * hat.abs(), dtype, "h")
    zero = torch.zeros(4, 1000, dtype=dtype, device=dev)                       # a row of zeros
    assert (ops.residual_norm(zero, zero, kind="rms", pre_weight=one, post_weight=one)[1] == 0).all()


def test_partial_gradients(dev):
    """Only some outputs or inputs take part: one of the two results, weights without inputs, inputs without weights."""
    from ddl import ops
    x, y, w = (rnd(dev, torch.float32, 9, 64, seed=s) for s in (1, 2, 3))
    w = w[0]
    for use in ("r", "h"):
        X, Y, W = (t.clone().requires_grad_(True) for t in (x, y, w))
        r, h = ops.residual_norm(X, Y, pre_weight=W, post_weight=W, gate=W, scale=0.7)
        a = torch.autograd.grad((r if use == "r" else h).sin().sum(), (X, Y, W))
        Xd, Yd = (t.double().requires_grad_(True) for t in (x, y))
        per_row = [w.double().expand(9, 64).clone().requires_grad_(True) for _ in range(3)]        # each use of w, row by row
        rd, hd = oracle.residual_norm(Xd, Yd, pre_weight=per_row[0], post_weight=per_row[1], gate=per_row[2], scale=0.7)
        b = torch.autograd.grad((rd if use == "r" else hd).sin().sum(), [Xd, Yd] + per_row, allow_unused=True)
        terms = torch.cat([g for g in b[2:] if g is not None])
        # a normalised value is off by at most 90 EPS of its size (hat_bound), the backward formula by three times that of the
        # largest term, and cos(r) of the outer function by once more: 1000 EPS of the terms' sizes covers the sum
        for got, want, size in zip(a, (b[0], b[1], terms.sum(0)), (b[0].abs() + 1, b[1].abs() + 1, terms.abs().sum(0) + 1)):
            assert ((got.double() - want).abs() <= 1000 * EPS * size * w.abs().max().item()).all()
    for leaf in range(3):
        a = [rnd(dev, torch.float32, 40, 24, seed=1), rnd(dev, torch.float32, 16, 24, seed=2), rnd(dev, torch.float32, 16, seed=3)]
        a[leaf].requires_grad_(True)
        (got,) = torch.autograd.grad(ops.linear(*a, activation="gelu").sum(), a[leaf])
        d = [t.detach().double() for t in a]
        d[leaf].requires_grad_(True)
        (want,) = torch.autograd.grad(oracle.linear(*d, act="gelu").sum(), d[leaf])
        torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)


def test_gradients_against_differences(dev):
    """The block as it is used, in fp32: directional derivatives against central differences of the 64-bit block."""
    from ddl import ops
    F, C, M = 40, 24, 50
    key = torch.tensor(KEYS[1], device=dev)
    p = dict(x=rnd(dev, torch.float32, M, C, seed=1), n=1 + 0.1 * rnd(dev, torch.float32, C, seed=2),
             g=rnd(dev, torch.float32, F, C, seed=3, scale=0.2), u=rnd(dev, torch.float32, F, C, seed=4, scale=0.2),
             d=rnd(dev, torch.float32, C, F, seed=5, scale=0.2), b=rnd(dev, torch.float32, C, seed=6), s=rnd(dev, torch.float32, C, seed=7))

    def block(o, drop, v):
        x, h = o.residual_norm(v["x"], kind="layer", pre_weight=v["n"])
        y = o.linear(o.gated_linear(h, v["g"], v["u"]) if o is ops else o.gated(h, v["g"], v["u"]), v["d"], v["b"])
        return o.residual_norm(x, drop(y), kind="layer", pre_weight=v["n"], gate=v["s"], scale=0.5)

    leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    r, h = block(ops, lambda y: ops.dropout(y, 0.3, key), leaves)
    grads = dict(zip(leaves, torch.autograd.grad((r.sin() + h).sum(), list(leaves.values()))))
    keep = torch.from_numpy(oracle.kept(KEYS[1], M * C, 0.3)).to(dev).double().view(M, C) / 0.7

    def loss(v):
        r, h = block(oracle, lambda y: y * keep, v)
        return (r.sin() + h).sum().item()

    for name in p:
        d = {k: v.double() for k, v in p.items()}
        step = rnd(dev, torch.float64, *p[name].shape, seed=11)
        e = 1e-6
        up, down = loss({**d, name: d[name] + e * step}), loss({**d, name: d[name] - e * step})
        want, got = (up - down) / (2 * e), (grads[name].double() * step).sum().item()
        size = (grads[name].double() * step).abs().sum().item()
        assert abs(got - want) <= 1e-4 * size + 1e-4, (name, got, want)


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------------
def _block(ops, t, key):
    x, h = ops.residual_norm(t["x"], pre_weight=t["n"])
    y = ops.linear(ops.gated_linear(h, t["g"], t["u"]), t["d"], t["b"], activation="gelu")
    y = ops.dropout(y, 0.3, key)
    return ops.residual_norm(x, y, pre_weight=t["n"], post_weight=t["n"], gate=t["n"])


def _params(dev, dtype, M, C=64, F=200):
    return dict(x=rnd(dev, dtype, M, C, seed=1), n=rnd(dev, dtype, C, seed=2), g=rnd(dev, dtype, F, C, seed=3, scale=0.2),
                u=rnd(dev, dtype, F, C, seed=4, scale=0.2), d=rnd(dev, dtype, C, F, seed=5, scale=0.2), b=rnd(dev, dtype, C, seed=6))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_training_step(dev, dtype, M):
    """Forward and backward of the block in a graph, replayed with eager work between; two graphs interleaved; every replay bit-equal
    to the eager call on the same inputs."""
    from ddl import ops
    graphs = []
    for which in range(2):
        t = {k: v.requires_grad_(True) for k, v in _params(dev, dtype, M + which).items()}
        key = torch.tensor(KEYS[which], device=dev)

        def step(t=t, key=key):
            r, h = _block(ops, t, key)
            return (r, h) + torch.autograd.grad((r, h), list(t.values()), (torch.ones_like(r), torch.ones_like(h)))

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out, t, step))
    for turn in range(3):
        for g, _, t, _ in graphs:
            with torch.no_grad():
                for i, v in enumerate(t.values()):
                    v.copy_(rnd(dev, torch.float32, *v.shape, seed=50 * turn + i, scale=0.3).to(dtype))
        for g, _, _, _ in graphs:
            g.replay()
        wants = [step() for _, _, _, step in graphs]
        torch.cuda.synchronize()
        for (g, out, _, _), want in zip(graphs, wants):
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_and_determinism(dev):
    from ddl import ops
    streams = [torch.cuda.Stream() for _ in range(2)]
    ts = [{k: v.requires_grad_(True) for k, v in _params(dev, torch.bfloat16, 700 + i, 256, 1000).items()} for i in range(2)]
    key = torch.tensor(KEYS[1], device=dev)

    def step(t):
        r, h = _block(ops, t, key)
        return (r.detach(), h.detach()) + torch.autograd.grad((r, h), list(t.values()), (torch.ones_like(r), torch.ones_like(h)))

    want = [step(t) for t in ts]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, t in zip(streams, ts):
            with torch.cuda.stream(s):
                got.append(step(t))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_large_offsets(dev):
    """Results and operands beyond 2^31 elements."""
    from ddl import ops
    M, N = 66000, 32776
    x, w = rnd(dev, torch.bfloat16, M, 8, seed=1), rnd(dev, torch.bfloat16, N, 8, seed=2)
    y = ops.linear(x, w)
    for m in (0, 65530, M - 1):
        z, zerr = product_bounds(x[m:m + 1].double(), w.double(), None, "none")
        close(y[m:m + 1], z, zerr, torch.bfloat16, "y")
    w2 = rnd(dev, torch.bfloat16, 24, N, seed=3, scale=N ** -0.5)
    z = ops.linear(y, w2)                                              # reads beyond 2^31
    want, zerr = product_bounds(y[M - 3:].double(), w2.double(), None, "none")
    close(z[M - 3:], want, zerr, torch.bfloat16, "z")
    C = 16384
    v = torch.zeros(2 ** 17 + 3, C, dtype=torch.bfloat16, device=dev)
    v[-1] = rnd(dev, torch.bfloat16, C, seed=5)
    one = torch.ones(C, dtype=torch.bfloat16, device=dev)
    _, h = ops.residual_norm(v, pre_weight=one)
    assert torch.equal(h[-1:], ops.residual_norm(v[-1:], pre_weight=one)[1]) and (h[-2] == 0).all()


def test_refusals(dev):
    from ddl import ops
    x, w, b = rnd(dev, torch.float32, 4, 8), rnd(dev, torch.float32, 6, 8), rnd(dev, torch.float32, 6)
    key = torch.tensor([1, 2], device=dev)
    n = torch.ones(8, device=dev)
    bad = [
        lambda: ops.linear(x, w[:, :7]), lambda: ops.linear(x, w.bfloat16()), lambda: ops.linear(x, w.cpu()),
        lambda: ops.linear(x, w, b[:5]), lambda: ops.linear(x, w, b, residual=x), lambda: ops.linear(x.double(), w.double()),
        lambda: ops.linear(x, w, b, activation="tanh"), lambda: ops.linear(x.long(), w.long()), lambda: ops.linear(x, w[0]),
        lambda: ops.gated_linear(x, w, w[:5]), lambda: ops.gated_linear(x, w, w, b), lambda: ops.gated_linear(x, w, w, b, b[:3]),
        lambda: ops.dropout(x, 1.5, key), lambda: ops.dropout(x, -0.1, key), lambda: ops.dropout(x, float("nan"), key),
        lambda: ops.dropout(x, 0.5, key.cpu()), lambda: ops.dropout(x, 0.5, key[:1]), lambda: ops.dropout(x, 0.5, key.float()),
        lambda: ops.dropout(x, 0.5, key, residual=w), lambda: ops.DropoutRng(0, dev, stream=2 ** 15),
        lambda: ops.residual_norm(x), lambda: ops.residual_norm(x, gate=n, pre_weight=n), lambda: ops.residual_norm(x, x[:3]),
        lambda: ops.residual_norm(x, pre_weight=n, pre_bias=n), lambda: ops.residual_norm(x, x, kind="batch"),
        lambda: ops.residual_norm(x, x, pre_weight=n[:7]), lambda: ops.residual_norm(x, x, pre_weight=n, gate=n.half()),
        lambda: ops.residual_norm(x, x, pre_bias=n, kind="layer"), lambda: ops.residual_norm(x, x, gate=x[:2]),
        lambda: ops.residual_norm(x, x, eps=-1.0), lambda: ops.residual_norm(torch.ones(2, 16385, device=dev), pre_weight=torch.ones(16385, device=dev)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    # second derivatives are refused, not silently zero
    xg = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.linear(xg, w, activation="gelu").sum(), xg, create_graph=True)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("M,K,N", [(1, 256, 4), (1, 768, 64), (3, 40, 17), (32, 65, 33)])
def test_few_rows_round_a_gradient_once(dev, dtype, gated, M, K, N):
    """Two parts hold dz to u^2 of itself (fp16: to half its smallest step).  Beside that stand dz's own error, from those of z and of
    the activation, and the fp32 sum over at most 2 x 66 terms; dz's rounding to u is not among them."""
    from ddl import ops
    x, w, v = rnd(dev, dtype, M, K), rnd(dev, dtype, N, K, seed=1, scale=K ** -0.5), rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5)
    dy = rnd(dev, dtype, M, N, seed=3)
    leaves = [t.requires_grad_(True) for t in ((x, w, v) if gated else (x, w))]
    y = ops.gated_linear(x, w, v) if gated else ops.linear(x, w, activation="silu")
    got = torch.autograd.grad(y, leaves, dy)
    xd, wd, vd, dyd = (t.detach().double() for t in (x, w, v, dy))
    (z, zerr), (up, uerr) = product_bounds(xd, wd, None, "none"), product_bounds(xd, vd, None, "none")
    s = torch.sigmoid(z)
    slope = s * (1 + z * (1 - s))
    serr, aerr = 1.2 * zerr + 16 * EPS * (1 + z.abs()), 1.13 * zerr + 16 * EPS * z.abs()
    dz = [dyd * up * slope, dyd * z * s] if gated else [dyd * slope]
    err = [dyd.abs() * (up.abs() * serr + 1.13 * uerr), dyd.abs() * aerr] if gated else [dyd.abs() * serr]
    weights = [wd, vd] if gated else [wd]
    step = tiny(dtype) if dtype == torch.float16 else 0.0
    err = [e + (oracle.rounding(dtype) ** 2 + 160 * EPS) * d.abs() + step for e, d in zip(err, dz)]
    close(got[0], sum(d @ p for d, p in zip(dz, weights)), sum(e @ p.abs() for e, p in zip(err, weights)), dtype, "dx")
    for i, d in enumerate(dz):
        close(got[1 + i], d.T @ xd, err[i].T @ xd.abs(), dtype, f"dw {i}")


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
def test_few_rows_gradients_that_overflow(dev, dtype):
    """dz beyond the type's range stays an infinity (what rounding took off it is not another one of the other sign)."""
    from ddl import ops
    top = torch.finfo(dtype).max
    x, w = torch.ones(2, 8, device=dev, dtype=dtype, requires_grad=True), torch.ones(8, 8, device=dev, dtype=dtype, requires_grad=True)
    y = ops.gated_linear(x, w, w)                          # up 8, gate's slope 1: dg = 8 dy
    dx, dw = torch.autograd.grad(y, (x, w), torch.full_like(y, top))
    assert torch.isposinf(dx).all() and torch.isposinf(dw).all()


@pytest.mark.parametrize("M,K,N", [(2500, 4096, 2500), (2100, 2048, 4200), (2560, 4096, 2816)])
def test_large_products_repeat_bit_for_bit(dev, M, K, N):
    """Tiles that reach beyond the output are moved inside it: some results have two writers."""
    from ddl import ops
    x, w = (rnd(dev, torch.bfloat16, *s, seed=1).requires_grad_(True) for s in ((M, K), (N, K)))
    dy = rnd(dev, torch.bfloat16, M, N, seed=2)

    def step():
        y = ops.linear(x, w, activation="relu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)

    want = step()
    for _ in range(6):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [3, 130])
def test_one_tensor_in_several_places_and_a_graph_walked_twice(dev, dtype, M):
    from ddl import ops
    C = 40
    x, w = rnd(dev, dtype, M, C).requires_grad_(True), rnd(dev, dtype, C, C, seed=1, scale=C ** -0.5).requires_grad_(True)
    parts = [x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)]
    weights = [w.detach().clone().requires_grad_(True) for _ in range(3)]
    y = ops.linear(ops.gated_linear(x, w, w), w, residual=x)
    z = ops.linear(ops.gated_linear(parts[0], weights[0], weights[1]), weights[2], residual=parts[1])
    assert torch.equal(y, z)
    dy = torch.ones((), device=dev, dtype=dtype).expand(M, C)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(s, t) for s, t in zip(first, again))
    each = torch.autograd.grad(z, parts + weights, dy)
    u = oracle.rounding(dtype)
    for got, terms in zip(first, (each[:2], each[2:])):              # a sum of two or three rounds twice at most, in any order
        total, mag = sum(t.double() for t in terms), sum(t.double().abs() for t in terms)
        assert ((got.double() - total).abs() <= 2.1 * u * mag + tiny(dtype)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [2, 4, 7, 8, 9, 12, 13, 16, 17, 24, 25, 31, 33])
def test_every_count_of_few_rows(dev, dtype, M):
    """Row counts on both sides of each variant's limit, a width beyond one strip of columns and off every vector."""
    K, N = 2051, 77
    x, w, b = rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, N, K, seed=2, scale=K ** -0.5), rnd(dev, dtype, N, seed=3)
    for act in ("none", "silu"):
        check_linear(dev, dtype, x, w, b, act, None)
