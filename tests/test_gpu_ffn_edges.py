"""Calls of the feed-forward operators that their documentation allows and tests/test_gpu_ffn.py does not make: more than one operand
in an unusual layout, the explicit forward / backward pairs, sizes at the limits.  Bounds are those of tests/test_gpu_ffn.py.
"""
import pytest
import torch

import ffn_oracle as oracle
from test_gpu_ffn import EPS, IDS, TYPES, act_and_slope, check_gated, check_linear, close, product_bounds, rnd, slope_bound, tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    from ddl import ops
    ops.require_ext()
    return torch.device("cuda", 0)


@pytest.fixture(scope="module")
def ext(dev):
    from ddl import ops
    return ops.require_ext()


# ---- operands that need both a change of layout and padding ------------------------------------------------------------------
def strided(t, how):
    """t's values behind strides that a product cannot read in place"""
    if how == "transposed":
        return t.t().contiguous().t()
    wide = torch.empty(t.shape[0], 2 * t.shape[1], dtype=t.dtype, device=t.device)
    v = wide[:, ::2]
    v.copy_(t)
    return v


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("how", ["transposed", "every other column"])
@pytest.mark.parametrize("M", [1, 5, 32, 33, 90])
@pytest.mark.parametrize("K", [41, 56])
def test_all_operands_strided_at_once(dev, dtype, how, M, K):
    N = 40
    x, g, u = (rnd(dev, dtype, *s, seed=i, scale=c) for i, (s, c) in enumerate((((M, K), 1.0), ((N, K), 0.2), ((N, K), 0.2))))
    check_gated(dev, dtype, *(strided(t, how) for t in (x, g, u)), None, None, "gelu")
    check_linear(dev, dtype, strided(x, how), strided(g, how), None, "silu", strided(rnd(dev, dtype, M, N, seed=4), how))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [3, 32, 40, 200])
def test_explicit_pairs_with_strided_operands(dev, ext, dtype, M):
    """The pairs that the model's units call: strided tensors give the bits that contiguous ones give."""
    K, N = 41, 27
    x, g, u, dy = (rnd(dev, dtype, *s, seed=i) for i, s in enumerate(((M, K), (N, K), (N, K), (M, N))))
    silu = 2

    def both(x, g, u, dy):
        h, z = ext.gated_forward(x, g, u, None, None, silu, True)
        y, s = ext.linear_forward(x, g, None, None, silu, True)
        out = [h, y] + list(ext.gated_backward(dy, x, g, u, z, silu, True, True, True))
        out += list(ext.linear_backward(dy, x, g, s, silu, True, True, True))
        return out + list(ext.linear_backward(dy, x, g, None, 0, True, True, True))

    want = both(x, g, u, dy)
    for how in ("transposed", "every other column"):
        for got, w in zip(both(*(strided(t, how) for t in (x, g, u, dy))), want):
            assert torch.equal(got, w), how


def test_kept_sums_of_another_call_are_refused(dev, ext):
    """Also where nothing is summed (K = 0), so that the number of rows cannot be told from the number of elements."""
    for K in (0, 8):
        few, many, w = (torch.zeros(n, K, device=dev) for n in (3, 50, 7))
        dy = torch.zeros(50, 7, device=dev)
        _, z = ext.linear_forward(few, w, None, None, 2, True)
        _, zz = ext.gated_forward(few, w, w, None, None, 2, True)
        with pytest.raises(ValueError, match="kept"):
            ext.linear_backward(dy, many, w, z, 2, True, True, True)
        with pytest.raises(ValueError, match="kept"):
            ext.gated_backward(dy, many, w, w, zz, 2, True, True, True)
        with pytest.raises(ValueError, match="kept"):
            ext.gated_backward(dy[:3], few, w, w, z, 2, True, True, True)


def test_dual_tensors_are_refused(dev):
    """No leaf requires a gradient, so no autograd node stands in the way: the result would have no tangent."""
    import torch.autograd.forward_ad as fwd
    from ddl import ops
    x, w = rnd(dev, torch.float32, 40, 8), rnd(dev, torch.float32, 8, 8, seed=1)
    key, v = torch.tensor([1, 2], device=dev), torch.ones(8, device=dev)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.linear(d, w), lambda: ops.linear(x, w, residual=d), lambda: ops.gated_linear(d, w, w),
                     lambda: ops.dropout(d, 0.5, key), lambda: ops.residual_norm(d, pre_weight=v), lambda: ops.residual_norm(x, d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # a dual gradient of an ordinary result
        leaf = x.clone().requires_grad_(True)
        for y in (ops.linear(leaf, w, activation="silu"), ops.gated_linear(leaf, w, w), ops.dropout(leaf, 0.5, key),
                  ops.residual_norm(leaf, pre_weight=v)[1]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, d)


# ---- large tiles, values -----------------------------------------------------------------------------------------------------
# (gated, M, K, N) -> (tile rows, tile columns, splits) of the forward product, d_x and d_w in 16 bits.  Together: both large tiles as
# single and as dual products, with one and two contraction segments, split and whole, with k starting elsewhere on each XCD (sizes of
# whole tiles and slabs), with tiles moved back inside off every vector (N % 8 = 4, odd), and slabs that end inside.
LARGE = {
    (False, 2560, 4096, 2816): [(128, 256, 1), (256, 256, 1), (256, 256, 1)],
    (False, 2100, 2048, 4200): [(256, 256, 1), (128, 256, 1), (256, 256, 1)],
    (False, 2500, 2500, 2501): [(128, 256, 1), (128, 256, 1), (128, 256, 1)],
    (False, 3001, 2052, 2052): [(128, 256, 1), (128, 256, 1), (128, 256, 1)],
    (False, 4001, 200, 3977): [(256, 256, 1), (32, 128, 1), (32, 128, 1)],
    (False, 4001, 200, 3980): [(256, 256, 1), (32, 128, 1), (32, 128, 1)],
    (True, 2048, 1024, 4096): [(256, 128, 1), (128, 256, 4), (128, 256, 1)],
    (True, 2011, 1000, 2708): [(256, 128, 1), (128, 256, 4), (128, 256, 1)],
    (True, 1500, 1030, 2300): [(128, 128, 1), (128, 256, 4), (128, 256, 1)],
    (True, 2051, 1100, 2051): [(256, 128, 1), (128, 256, 2), (128, 256, 1)],
    (True, 2560, 2048, 2560): [(256, 128, 1), (128, 256, 1), (256, 256, 1)],
    (True, 2500, 2052, 2052): [(256, 128, 1), (128, 256, 1), (256, 256, 1)],
}


def check_kept_sums(dev, ext, dtype, gated, M, K, N, bias):
    """What the forward pass keeps: the fp32 sums themselves, element for element."""
    x, b = rnd(dev, dtype, M, K, seed=1), rnd(dev, dtype, N, seed=4) if bias else None
    w = [rnd(dev, dtype, N, K, seed=2 + i, scale=K ** -0.5) for i in range(1 + gated)]
    z = (ext.gated_forward(x, *w, b, b, 2, True) if gated else ext.linear_forward(x, *w, b, None, 2, True))[1]
    assert z.shape[:2] == (1 + gated, M) and z.dtype == torch.float32
    for plane, v in zip(z, w):
        want, bound = product_bounds(x.double(), v.double(), b.double() if bias else None, "silu")
        assert ((plane[:, :N].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("case", list(LARGE), ids=str)
def test_large_tiles(dev, ext, dtype, case):
    gated, M, K, N = case
    name = "bf16" if dtype == torch.bfloat16 else "fp16"
    assert [ext.product_plan(what, name, M, K, N, gated) for what in ("forward", "dx", "dw")] == LARGE[case]
    bias = N % 3 > 0
    check_kept_sums(dev, ext, dtype, gated, M, K, N, bias)
    x, w = rnd(dev, dtype, M, K, seed=1), [rnd(dev, dtype, N, K, seed=2 + i, scale=K ** -0.5) for i in range(1 + gated)]
    b = [rnd(dev, dtype, N, seed=4 + i) if bias else None for i in range(1 + gated)]
    if gated:
        check_gated(dev, dtype, x, *w, *b, "gelu")
    else:
        check_linear(dev, dtype, x, *w, *b, "gelu", rnd(dev, dtype, M, N, seed=6))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("M,K,N", [(5, 40, 19), (70, 41, 23), (300, 200, 260), (900, 300, 1203), (1500, 200, 2052),
                                   (2049, 100, 4101)])
def test_kept_sums(dev, ext, dtype, gated, M, K, N):
    check_kept_sums(dev, ext, dtype, gated, M, K, N, bias=True)


# ---- residual_norm -----------------------------------------------------------------------------------------------------------
def test_strided_norm_inputs_are_copied_once(dev):
    """A step on strided rows makes one copy of each of them more than a step on contiguous rows, and gives the same bits."""
    from ddl import ops
    x, y, gate, dr, dh = (rnd(dev, torch.float32, 50, 64, seed=i) for i in range(5))
    w = rnd(dev, torch.float32, 64, seed=6).requires_grad_(True)

    def step(how):
        leaves = [(strided(t, "transposed") if how else t.clone()).requires_grad_(True) for t in (x, y, gate)]
        made = torch.cuda.memory_stats()["allocation.all.allocated"]
        outs = ops.residual_norm(leaves[0], leaves[1], kind="layer", pre_weight=w, post_weight=w, gate=leaves[2])
        grads = torch.autograd.grad(outs, leaves + [w], (dr, dh))
        return torch.cuda.memory_stats()["allocation.all.allocated"] - made, [o.detach() for o in outs] + list(grads)

    step(False)
    plain, want = step(False)
    copies, got = step(True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert copies - plain == 3
    r, h = ops.residual_norm(strided(x, "transposed"), pre_weight=w.detach())
    assert torch.equal(h, ops.residual_norm(x, pre_weight=w.detach())[1]) and not r.is_contiguous()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_channel_gate_beside_a_single_row(dev, dtype):
    from ddl import ops
    x, y, dr, dh = (rnd(dev, dtype, 72, seed=i) for i in range(4))
    for ptype in {dtype, torch.float32}:
        g, w = (rnd(dev, ptype, 72, seed=i).requires_grad_(True) for i in (5, 6))
        X, Y = (t.clone().requires_grad_(True) for t in (x, y))
        one = ops.residual_norm(X, Y, gate=g, pre_weight=w)
        two = ops.residual_norm(X[None], Y[None], gate=g, pre_weight=w)
        a = torch.autograd.grad(one, (X, Y, g, w), (dr, dh))
        b = torch.autograd.grad(two, (X, Y, g, w), (dr[None], dh[None]))
        assert all(torch.equal(p, q[0]) for p, q in zip(one, two)) and all(torch.equal(p, q) for p, q in zip(a, b))


# ---- many rows -----------------------------------------------------------------------------------------------------------------
def test_more_rows_than_one_line_of_workgroups(dev):
    """A launch has fewer than 2^32 threads and 65536 workgroups along x here: all rows are reached, also where each has a workgroup."""
    from ddl import ops
    for dtype, M, C in ((torch.float16, 2 ** 26 + 5, 4), (torch.bfloat16, 70003, 4104), (torch.float32, 65537, 16384)):
        w = rnd(dev, dtype, C, seed=2).requires_grad_(True)
        x = torch.zeros(M, C, dtype=dtype, device=dev)
        some = torch.tensor([0, 1, 65535, 65536, M // 2, M - 2, M - 1], device=dev)
        x[some] = rnd(dev, dtype, 7, C, seed=1)
        x.requires_grad_(True)
        _, h = ops.residual_norm(x, pre_weight=w)
        part = x.detach()[some].requires_grad_(True)
        _, want = ops.residual_norm(part, pre_weight=w)
        others = torch.ones(M, dtype=torch.bool, device=dev).index_fill_(0, some, False)
        assert torch.equal(h[some], want) and not (h.any(1) & others).any()
        dh = torch.zeros_like(h)
        dh[some] = 1
        (dx,) = torch.autograd.grad(h, x, dh)
        assert torch.equal(dx[some], torch.autograd.grad(want, part, torch.ones_like(want))[0])
        assert not (dx.any(1) & others).any()


def test_products_of_many_rows(dev):
    from ddl import ops
    M = 2 ** 28 + 3
    x, w = torch.zeros(M, 8, dtype=torch.bfloat16, device=dev), rnd(dev, torch.bfloat16, 8, 8, seed=1)
    some = torch.tensor([0, 1, 2 ** 27, M - 2, M - 1], device=dev)
    x[some] = rnd(dev, torch.bfloat16, 5, 8, seed=2)
    y = ops.linear(x, w)
    want, bound = product_bounds(x[some].double(), w.double(), None, "none")
    close(y[some], want, bound, torch.bfloat16, "y")
    assert (y[2:2 ** 27] == 0).all()


def test_widths_beyond_the_limit_are_refused(dev):
    """Nothing is allocated: the weights have no columns, or no rows."""
    from ddl import ops
    wide = 2 ** 26 + 1
    with pytest.raises(ValueError, match="columns"):
        ops.linear(torch.empty(1, 0, device=dev), torch.empty(wide, 0, device=dev))
    with pytest.raises(ValueError, match="columns"):
        ops.gated_linear(torch.empty(0, wide, device=dev), torch.empty(0, wide, device=dev), torch.empty(0, wide, device=dev))


def test_far_sums(dev):
    from test_ffn_ops import check_far_sums
    check_far_sums(dev)


def test_a_key_in_any_layout(dev):
    """Two int64 values, as on the CPU: a column of a table, a [2, 1] tensor, one value for both."""
    from ddl import ops
    x, k = rnd(dev, torch.float32, 40, 30), torch.tensor([7, 9], device=dev)
    want = ops.dropout(x, 0.5, k)
    table = torch.stack([k, k + 1], 1)
    for key in (table[:, 0], k.view(2, 1), table[:, :1]):
        leaf = x.clone().requires_grad_(True)
        y = ops.dropout(leaf, 0.5, key)
        assert torch.equal(y, want)
        (dx,) = torch.autograd.grad(y, leaf, x)
        assert torch.equal(dx, want)
    same = torch.tensor(7, device=dev).expand(2)
    assert torch.equal(ops.dropout(x, 0.5, same), ops.dropout(x, 0.5, same.contiguous()))


# ---- fp16: dz outside the type's range, gradients inside ----------------------------------------------------------------------
def gradient_bounds(x, w, b, act, dy, dtype):
    """(dz of each weight, its bound) in 64 bits.  dz is held rounded to `dtype` times a power of two 2^e: off by half a step, u of itself,
    or 2^-25 2^e in fp16 where it is small; 2^e is at most 2^-14 of the largest unless that lies in [2^-8, 65504], where it is 1."""
    X, W, B, D = x.double(), [t.double() for t in w], None if b is None else b.double(), dy.double()
    z, zerr = product_bounds(X, W[0], B, act)
    a, da = act_and_slope(z, act)
    serr = slope_bound(z, zerr, act)
    if len(w) == 2:
        up, uerr = product_bounds(X, W[1], B, act)
        aerr = 1.13 * zerr + 16 * EPS * (a.abs() + z.abs())
        dz = [D * up * da, D * a]
        e32 = [D.abs() * (serr * (up.abs() + uerr) + da.abs() * uerr) + 8 * EPS * dz[0].abs(), D.abs() * aerr + 8 * EPS * dz[1].abs()]
    else:
        dz = [D * da]
        e32 = [D.abs() * serr + 4 * EPS * dz[0].abs()]
    top, u = max(d.abs().max().item() for d in dz), oracle.rounding(dtype)
    step = tiny(dtype) if 2.0 ** -8 <= top <= 65504 else 2.0 ** -39 * top
    return dz, [e + u * (d.abs() + e) + step for d, e in zip(dz, e32)], top


def check_gradients(ops, x, w, b, act, dy, dtype, got):
    dz, err, top = gradient_bounds(x, w, b, act, dy, dtype)
    M, N = dy.shape
    X, W = x.double(), [t.double() for t in w]
    size = sum(d.abs() @ v.abs() for d, v in zip(dz, W))
    want = [sum(d @ v for d, v in zip(dz, W))] + [d.T @ X for d in dz]
    bound = [sum(e @ v.abs() for e, v in zip(err, W)) + (2 * N + 16) * EPS * size]
    bound += [e.T @ X.abs() + (M + 16) * EPS * (d.abs().T @ X.abs()) for d, e in zip(dz, err)]
    for t, v, e, what in zip(got, want, bound, ("dx", "dw 0", "dw 1")):
        assert v.abs().max() + e.max() < 65504, f"{what} itself is out of range"
        close(t, v, e, dtype, what)
    return top


#: scales of x, w_gate (or w), w_up, dy; the range of the largest |dz|
RANGES = {"beyond": ((0.01, 1e-3, 1e4, 300.0), (65504, 1e9)), "below": ((100.0, 1e-3, 1e-3, 2e-6), (1e-9, 2.0 ** -13)),
          "inside": ((1.0, 0.1, 0.1, 1.0), (2.0 ** -8, 65504))}


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("where", list(RANGES))
@pytest.mark.parametrize("M", [1, 5, 32, 33, 300, 2500])
def test_gradients_of_dz_out_of_range(dev, dtype, where, M):
    from ddl import ops
    K, N = (64, 72) if M < 2500 else (1024, 2052)
    (sx, sg, su, sd), (lo, hi) = RANGES[where]
    if where == "beyond" and M > 32:
        sx *= (32 / M) ** 0.5                                          # d_w, a sum over M rows, has to stay in range itself
    fan = (64 / K) ** 0.5                                              # the sums of the small case, also at K = 1024
    x, dy = rnd(dev, dtype, M, K, seed=1, scale=sx), rnd(dev, dtype, M, N, seed=2, scale=sd)
    g, u = rnd(dev, dtype, N, K, seed=3, scale=sg * fan), rnd(dev, dtype, N, K, seed=4, scale=su * fan)
    leaves = [t.requires_grad_(True) for t in (x, g, u)]
    got = torch.autograd.grad(ops.gated_linear(*leaves), leaves, dy)
    top = check_gradients(ops, x.detach(), [g.detach(), u.detach()], None, "silu", dy, dtype, got)
    assert M == 1 or lo <= top <= hi
    # one weight: only the slope, up to 1.1, stands between dy and dz
    b = torch.full((N,), 2.4, device=dev, dtype=dtype)
    dy = (rnd(dev, torch.float32, M, N, seed=5).sign() * {"beyond": 65000.0, "below": 2e-6, "inside": 1.0}[where]).to(dtype)
    v = (g.detach() * (1e-3 if where == "beyond" else 1.0)).to(dtype).requires_grad_(True)
    xs = (x.detach() * (0.1 if where == "beyond" else 1.0)).to(dtype).requires_grad_(True)
    got = torch.autograd.grad(ops.linear(xs, v, b, activation="silu"), (xs, v), dy)
    check_gradients(ops, xs.detach(), [v.detach()], b, "silu", dy, dtype, got)


@pytest.mark.parametrize("M", [8, 90])
def test_captured_gradients_follow_the_range(dev, M):
    """The power of two is chosen on the device: replays of one graph see ordinary, huge and tiny gradients in turn."""
    from ddl import ops
    x, g, u = (rnd(dev, torch.float16, *s, seed=i, scale=c).requires_grad_(True)
               for i, (s, c) in enumerate((((M, 64), 0.01), ((72, 64), 1e-3), ((72, 64), 1e4))))
    dy = torch.empty(M, 72, dtype=torch.float16, device=dev)

    def step():
        return torch.autograd.grad(ops.gated_linear(x, g, u), (x, g, u), dy)

    dy.fill_(1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, scale in enumerate((1.0, 300.0, 1e-6, 300.0, 1.0)):
        dy.copy_(rnd(dev, torch.float16, M, 72, seed=20 + i, scale=scale))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        check_gradients(ops, x.detach(), [g.detach(), u.detach()], None, "silu", dy, torch.float16, out)


def test_infinite_gradients_stay_infinite(dev):
    """An infinity or NaN in dy stays where the formula has it, whatever the scale the others are held in."""
    from ddl import ops
    for M in (6, 60):
        for scale in (1.0, 3e4):
            x, w = (rnd(dev, torch.float16, *s, seed=i, scale=0.01).requires_grad_(True) for i, s in enumerate(((M, 64), (72, 64))))
            b = torch.full((72,), 2.4, device=dev, dtype=torch.float16)
            dy = rnd(dev, torch.float16, M, 72, seed=3).sign() * scale
            y = ops.linear(x, w, b, activation="silu")
            want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
            dy[2, 5], dy[3, 7] = float("inf"), float("nan")
            dx, dw = torch.autograd.grad(y, (x, w), dy)
            rows, cols = ([i for i in range(n) if i not in bad] for n, bad in ((M, (2, 3)), (72, (5, 7))))
            assert torch.equal(dx[rows], want[0][rows]) and torch.equal(dw[cols], want[1][cols])
            assert dx[2].isinf().all() and dx[3].isnan().all() and dw[5].isinf().all() and dw[7].isnan().all()


# ---- tensors whose memory does not hold their values -----------------------------------------------------------------------------
def test_negated_views(dev):
    """The imaginary part of a conjugate is a lazily negated view: every operator sees its values, in every place, gradients as well."""
    from ddl import ops

    def negated(t):
        v = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v

    key = torch.tensor([1, 2], device=dev)
    for M in (5, 50):
        x, y, res = (rnd(dev, torch.float32, M, 24, seed=i) for i in range(3))
        w, v = rnd(dev, torch.float32, 24, 24, seed=4), rnd(dev, torch.float32, 24, seed=5)
        calls = [lambda x, y, res, w, v: [ops.linear(x, w, v, activation="silu", residual=res)],
                 lambda x, y, res, w, v: [ops.gated_linear(x, w, w, v, v)],
                 lambda x, y, res, w, v: [ops.dropout(x, 0.3, key, residual=res)],
                 lambda x, y, res, w, v: ops.residual_norm(x, y, kind="layer", pre_weight=v, pre_bias=v, post_weight=v, post_bias=v, gate=v),
                 lambda x, y, res, w, v: ops.residual_norm(x, y, gate=res, pre_weight=v)]
        for i, call in enumerate(calls):
            results = []
            for view in (lambda t: t.clone(), negated):
                with torch.no_grad():
                    results.append(list(call(*(view(t) for t in (x, y, res, w, v)))))
                leaves = [view(t).detach().requires_grad_(True) for t in (x, y, res, w, v)]
                outs = call(*leaves)
                grads = torch.autograd.grad(outs, leaves, [view(x) for _ in outs], allow_unused=True)
                results[-1] += [g for g in grads if g is not None]
            assert len(results[0]) == len(results[1])
            assert all(torch.equal(a, b) for a, b in zip(*results)), i


# ---- captures ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("op", ["linear", "gated_linear", "dropout", "residual_norm"])
def test_a_captured_backward_beside_an_eager_result(dev, op):
    """An eager result of the leaf on the default stream is alive: the captured backward pass raises instead of ending the process,
    and works once the result is gone."""
    from ddl import ops
    x, w = rnd(dev, torch.float32, 40, 16).requires_grad_(True), rnd(dev, torch.float32, 16, 16, seed=1).requires_grad_(True)
    key = torch.tensor([1, 2], device=dev)
    call = {"linear": lambda x: ops.linear(x, w, activation="silu"), "gated_linear": lambda x: ops.gated_linear(x, w, w),
            "dropout": lambda x: ops.dropout(x, 0.3, key), "residual_norm": lambda x: ops.residual_norm(x, pre_weight=w[0].detach())[1]}[op]
    dy = rnd(dev, torch.float32, 40, 16, seed=2)
    (want,) = torch.autograd.grad(call(x), x, dy)
    held = call(x)                                                   # x's accumulation node stays on the default stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(x)
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(y, x, dy)
    del y, held, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dx,) = torch.autograd.grad(call(x), x, dy)
    for _ in range(3):
        graph.replay()
        assert torch.equal(dx, want)
        (again,) = torch.autograd.grad(call(x), x, dy)
        assert torch.equal(again, want)
