"""Cases of the feed-forward operators (``ddl.ops``): ``linear``, ``gated_linear``, ``dropout``, ``residual_norm``.

``run`` computes a case either in plain form (elementary torch operations in 32 bits, rounded once at the end) or, with
``own`` set, through the framework's entry points, as a training or serving program calls them.

* ``linear``:         y = act(x W^T + b) + residual
* ``gated_linear``:   h = act(x Wg^T + bg) * (x Wu^T + bu)
* ``dropout``:        y = residual + x * keep / (1 - p); keep comes from the counter-based generator Philox4x32 (Salmon et
                      al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with seven rounds, so no mask is stored:
                      word e % 4 of block (e // 4, call) under the key ``seed`` decides element e, dropped below p * 2^32
* ``residual_norm``:  r = x + scale * gate * post(branch), h = pre(r); post / pre: layer or RMS norm with its weights

A training case returns the outputs and every gradient; the other cases are inference.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")


# ---- the cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the classifier of one image at inference: 1024 pooled features -> 5 classes; nothing but latency
        dict(name="linear one image", op="linear", rows=1, k=1024, n=5, dtype="fp32", act="none", bias=True, residual=False,
             train=False),
        # hidden layer of a classifier head on the default batch of 30, fp32 as the framework trains by default
        dict(name="linear head step", op="linear", rows=30, k=1024, n=4096, dtype="fp32", act="gelu", bias=True,
             residual=False, train=True),
        # sizes that fit no tile, rows that are not 16-byte aligned
        dict(name="linear ragged step", op="linear", rows=777, k=1021, n=1531, dtype="fp16", act="silu", bias=True,
             residual=True, train=True),
        # output projection of a wide block with its residual, a training step over 8192 rows
        dict(name="linear large step", op="linear", rows=8192, k=4096, n=4096, dtype="bf16", act="gelu", bias=True,
             residual=True, train=True),
        # a single token through a wide gated block: every weight is read once for one row
        dict(name="gated one token", op="gated", rows=1, k=4096, n=11264, dtype="bf16", act="silu", bias=False,
             train=False),
        # gated head on 128 images, fp32
        dict(name="gated head step", op="gated", rows=128, k=1024, n=4096, dtype="fp32", act="silu", bias=True,
             train=True),
        # ragged rows and widths with biases
        dict(name="gated ragged step", op="gated", rows=2011, k=1000, n=2708, dtype="bf16", act="gelu_tanh", bias=True,
             train=True),
        # the largest training step
        dict(name="gated large step", op="gated", rows=8192, k=4096, n=8192, dtype="bf16", act="silu", bias=False,
             train=True),
        # pooled features of the default batch
        dict(name="dropout features", op="dropout", rows=30, k=1024, dtype="fp32", p=0.2, residual=False, train=True),
        # a branch that joins its residual stream, a long training step
        dict(name="dropout large", op="dropout", rows=16384, k=8192, dtype="bf16", p=0.1, residual=True, train=True),
        # a single token between two blocks
        dict(name="norm one token", op="norm", rows=1, k=4096, dtype="bf16", kind="rms", post=True, pre=True,
             gate="channel", scale=1.0, bias=False, train=False),
        # a training step between two wide blocks
        dict(name="norm large step", op="norm", rows=16384, k=4096, dtype="bf16", kind="layer", post=True, pre=True,
             gate="channel", scale=0.5, bias=True, train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "gated", "dropout", "norm"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("linear", "gated"):
        most = 4.0e11 if op == "linear" else 8.0e11
        if dtype == "fp32":
            most /= 8
        while True:
            rows, k, n = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 5 if op == "linear" else 64, 12288)
            if rng.random() < 0.6:                      # widths as models have them; the others are odd as they come
                k, n = max(64, k // 64 * 64), max(8, n // 64 * 64)
            flops = 2.0 * rows * k * n * (1 if op == "linear" else 2)
            if flops <= most:
                break
        case = dict(op=op, rows=rows, k=k, n=n, dtype=dtype, bias=rng.random() < 0.5, train=rng.random() < 0.6)
        if op == "linear":
            case.update(act=rng.choice(ACTIVATIONS), residual=rng.random() < 0.5)
        else:
            case.update(act=rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid", "relu"]))
        return case
    rows, k = _log(rng, 1, 16384), _log(rng, 16, 8192)
    if rng.random() < 0.6:
        k = max(16, k // 16 * 16)
    if op == "dropout":
        return dict(op=op, rows=rows, k=k, dtype=dtype, p=rng.choice([0.05, 0.1, 0.2, 0.5, 0.9]),
                    residual=rng.random() < 0.5, train=rng.random() < 0.7)
    post, pre = rng.choice([(True, True), (True, False), (False, True)])
    return dict(op=op, rows=rows, k=k, dtype=dtype, kind=rng.choice(["rms", "layer"]), post=post, pre=pre,
                gate=rng.choice(["none", "channel", "full"]), scale=rng.choice([1.0, 0.5]), bias=rng.random() < 0.5,
                train=rng.random() < 0.6)


def _inputs(case, seed, device):
    """Named inputs of a case, from the seed alone."""
    g = torch.Generator(device=device).manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    rows, k, op = case["rows"], case["k"], case["op"]

    def rnd(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=device) * scale + shift).to(dt)

    t = {"x": rnd(rows, k)}
    if op == "linear":
        n = case["n"]
        t["w"] = rnd(n, k, scale=k ** -0.5)
        t["b"] = rnd(n, scale=0.1) if case["bias"] else None
        t["residual"] = rnd(rows, n) if case["residual"] else None
        t["dy"] = rnd(rows, n) if case["train"] else None
    elif op == "gated":
        n = case["n"]
        t["wg"], t["wu"] = rnd(n, k, scale=k ** -0.5), rnd(n, k, scale=k ** -0.5)
        t["bg"], t["bu"] = (rnd(n, scale=0.1), rnd(n, scale=0.1)) if case["bias"] else (None, None)
        t["dy"] = rnd(rows, n) if case["train"] else None
    elif op == "dropout":
        t["residual"] = rnd(rows, k) if case["residual"] else None
        t["dy"] = rnd(rows, k) if case["train"] else None
        t["key"] = torch.randint(0, 2 ** 62, (2,), generator=g, device=device)
    else:
        t["branch"] = rnd(rows, k, scale=2.0, shift=0.25)
        t["gate"] = {"none": None, "channel": rnd(k, scale=0.3, shift=0.5), "full": rnd(rows, k, scale=0.5)}[case["gate"]]
        for name in ("post", "pre"):
            on = case[name]
            t[name + "_w"] = rnd(k, scale=0.2, shift=1.0) if on else None
            t[name + "_b"] = rnd(k, scale=0.2) if on and case["bias"] and case["kind"] == "layer" else None
        t["dr"] = rnd(rows, k) if case["train"] else None
        t["dh"] = rnd(rows, k) if case["train"] and case["pre"] else None
    return t


#: the inputs a training case has gradients for, in the order they are returned
LEAVES = {"linear": ("x", "w", "b", "residual"), "gated": ("x", "wg", "wu", "bg", "bu"), "dropout": ("x", "residual"),
          "norm": ("x", "branch", "gate", "post_w", "post_b", "pre_w", "pre_b")}


def prepare(case, seed):
    t = _inputs(case, seed, "cuda")
    if case["train"]:
        for name in LEAVES[case["op"]]:
            if t[name] is not None:
                t[name].requires_grad_(True)
    return dict(case=case, **t)


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _own(s):
    from ddl import ops

    c = s["case"]
    op = c["op"]
    if op == "linear":
        outs = (ops.linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["residual"]),)
    elif op == "gated":
        outs = (ops.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["act"]),)
    elif op == "dropout":
        outs = (ops.dropout(s["x"], c["p"], s["key"], residual=s["residual"]),)
    else:
        r, h = ops.residual_norm(s["x"], s["branch"], kind=c["kind"], eps=1e-6, pre_weight=s["pre_w"], pre_bias=s["pre_b"],
                                 post_weight=s["post_w"], post_bias=s["post_b"], gate=s["gate"], scale=c["scale"])
        outs = (r,) if h is None else (r, h)
    grads = ()
    if c["train"]:
        leaves = [s[n] for n in LEAVES[op] if s[n] is not None]
        douts = [s["dy"]] if op != "norm" else [d for d in (s["dr"], s["dh"]) if d is not None]
        grads = torch.autograd.grad(outs, leaves, douts)
    return _named(c, s, outs, grads)


def _named(c, s, outs, grads):
    got = {"out%d" % i: o for i, o in enumerate(outs)}
    if grads:
        got.update(zip(["d_" + n for n in LEAVES[c["op"]] if s[n] is not None], grads))
    return got


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    sig = 1 / (1 + torch.exp(-z))
    return (sig, sig * (1 - sig)) if act == "sigmoid" else (z * sig, sig * (1 + z * (1 - sig)))


def _keep(key, count, p):
    """Which of ``count`` elements stay: Philox4x32 with seven rounds, in 64-bit integers."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 3) // 4, device=key.device, dtype=torch.int64)
    seed, call = key[0], key[1]
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = (call & low).expand_as(block), ((call >> 32) & low).expand_as(block)
    k0, k1 = seed & low, (seed >> 32) & low

    def turn(c0, c1, c2, c3, k0, k1):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        return ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low

    for i in range(7):
        c0, c1, c2, c3 = turn(c0, c1, c2, c3, (k0 + i * 0x9E3779B9) & low, (k1 + i * 0xBB67AE85) & low)
    words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:count]
    return words >= int(p * 2 ** 32)


def _norm(v, w, b, kind):
    """(n, vhat, rstd): the normalised rows with and without the weights."""
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6)
    hat = c * rstd
    n = hat * w
    return n if b is None else n + b, hat, rstd


def _norm_back(dn, hat, rstd, w, kind):
    g = dn * w
    g_mean = g.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (g - g_mean - hat * (g * hat).mean(1, keepdim=True))


def _plain(s):
    c = s["case"]
    op, train, dt = c["op"], c["train"], s["x"].dtype
    f = {n: t.detach().float() if isinstance(t, torch.Tensor) and n != "key" else t for n, t in s.items()}
    x, grads = f["x"], []
    if op == "linear":
        z = x @ f["w"].T
        z = z if f["b"] is None else z + f["b"]
        a, da = _act(z, c["act"])
        outs = [a if f["residual"] is None else a + f["residual"]]
        if train:
            dz = f["dy"] * da
            grads = [dz @ f["w"], dz.T @ x, dz.sum(0) if f["b"] is not None else None,
                     f["dy"] if f["residual"] is not None else None]
    elif op == "gated":
        g, u = x @ f["wg"].T, x @ f["wu"].T
        if f["bg"] is not None:
            g, u = g + f["bg"], u + f["bu"]
        a, da = _act(g, c["act"])
        outs = [a * u]
        if train:
            dg, du = f["dy"] * u * da, f["dy"] * a
            grads = [dg @ f["wg"] + du @ f["wu"], dg.T @ x, du.T @ x]
            grads += [dg.sum(0), du.sum(0)] if f["bg"] is not None else [None, None]
    elif op == "dropout":
        keep = _keep(s["key"], x.numel(), c["p"]).reshape(x.shape).to(torch.float32) * (1 / (1 - c["p"]))
        outs = [x * keep if f["residual"] is None else x * keep + f["residual"]]
        if train:
            grads = [f["dy"] * keep, f["dy"] if f["residual"] is not None else None]
    else:
        y = f["branch"]
        n, nhat, nrstd = _norm(y, f["post_w"], f["post_b"], c["kind"]) if c["post"] else (y, None, None)
        gate = c["scale"] if f["gate"] is None else f["gate"] * c["scale"]
        r = x + gate * n
        outs = [r]
        if c["pre"]:
            h, hat, rstd = _norm(r, f["pre_w"], f["pre_b"], c["kind"])
            outs.append(h)
        if train:
            dr = f["dr"]
            if c["pre"]:
                dr = dr + _norm_back(f["dh"], hat, rstd, f["pre_w"], c["kind"])
            dn = gate * dr
            dgate = None
            if f["gate"] is not None:
                dgate = c["scale"] * n * dr
                dgate = dgate.sum(0) if c["gate"] == "channel" else dgate
            dy = _norm_back(dn, nhat, nrstd, f["post_w"], c["kind"]) if c["post"] else dn
            grads = [dr, dy, dgate, (dn * nhat).sum(0) if c["post"] else None, dn.sum(0) if f["post_b"] is not None else None,
                     (f["dh"] * hat).sum(0) if c["pre"] else None, f["dh"].sum(0) if f["pre_b"] is not None else None]
    return _named(c, s, [o.to(dt) for o in outs], [g.to(dt) for g in grads if g is not None])


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    """The case from its formulas in 64 bits; gradients by differentiation of the formulas, not by the plain form's."""
    t = _inputs(case, seed, "cuda")
    d = {n: v.double() if v is not None and n != "key" else v for n, v in t.items()}
    leaves = [n for n in LEAVES[case["op"]] if d[n] is not None]
    for n in leaves:
        d[n].requires_grad_(case["train"])

    def act(z):
        if case["act"] == "gelu_tanh":
            return z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "sigmoid": torch.special.expit,
                "silu": lambda v: v * torch.special.expit(v), "gelu": lambda v: v * torch.special.ndtr(v)}[case["act"]](z)

    def lin(w, b):
        z = d["x"].matmul(w.t())
        return z if b is None else z + b

    def norm(v, w, b):
        if case["kind"] == "layer":
            v = v - v.sum(1, keepdim=True) / v.shape[1]
        n = v / (v.pow(2).sum(1, keepdim=True) / v.shape[1] + 1e-6).sqrt() * w
        return n if b is None else n + b

    op = case["op"]
    if op == "linear":
        y = act(lin(d["w"], d["b"]))
        outs = [y if d["residual"] is None else y + d["residual"]]
    elif op == "gated":
        outs = [act(lin(d["wg"], d["bg"])) * lin(d["wu"], d["bu"])]
    elif op == "dropout":
        y = d["x"] * _kept_in_integers(t["key"].tolist(), case["rows"] * case["k"], case["p"], d["x"]) / (1 - case["p"])
        outs = [y if d["residual"] is None else y + d["residual"]]
    else:
        n = norm(d["branch"], d["post_w"], d["post_b"]) if case["post"] else d["branch"]
        r = d["x"] + case["scale"] * (n if d["gate"] is None else d["gate"] * n)
        outs = [r] + ([norm(r, d["pre_w"], d["pre_b"])] if case["pre"] else [])
    grads = []
    if case["train"]:
        douts = [d["dy"]] if op != "norm" else [v for v in (d["dr"], d["dh"]) if v is not None]
        grads = torch.autograd.grad(outs, [d[n] for n in leaves], douts)
    got = {"out%d" % i: o.detach() for i, o in enumerate(outs)}
    got.update(zip(["d_" + n for n in leaves], grads))
    return got


def _kept_in_integers(key, count, p, like):
    """The kept elements as ones, from the generator's definition in unsigned numpy arithmetic."""
    import numpy as np

    m32 = np.uint64(0xFFFFFFFF)
    n = (count + 3) // 4
    i = np.arange(n, dtype=np.uint64)
    ctr = [i & m32, i >> np.uint64(32), np.full(n, key[1] & 0xFFFFFFFF, np.uint64), np.full(n, key[1] >> 32, np.uint64)]
    ks = [key[0] & 0xFFFFFFFF, key[0] >> 32]
    for _ in range(7):
        p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(p1 >> np.uint64(32)) ^ ctr[1] ^ np.uint64(ks[0]), p1 & m32, (p0 >> np.uint64(32)) ^ ctr[3] ^ np.uint64(ks[1]),
               p0 & m32]
        ks = [(ks[0] + 0x9E3779B9) % 2 ** 32, (ks[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(ctr, 1).reshape(-1)[:count]
    return torch.from_numpy((words >= np.uint64(int(p * 2 ** 32))).reshape(like.shape)).to(like.device).to(like.dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _flops(c):
    if c["op"] in ("linear", "gated"):
        return 2.0 * c["rows"] * c["k"] * c["n"] * (2 if c["op"] == "gated" else 1) * (3 if c["train"] else 1)
    return 8.0 * c["rows"] * c["k"]


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    rows, k, train = case["rows"], case["k"], case["train"]
    if case["op"] in ("linear", "gated"):
        n, two = case["n"], 2 if case["op"] == "gated" else 1
        params = two * n * k + (two * n if case["bias"] else 0)
        count = rows * k + params + rows * n + (rows * n if case.get("residual") else 0)
        if train:
            count += rows * n + rows * k + params       # dy in; dx and the weights' gradients out
    elif case["op"] == "dropout":
        count = rows * k * (3 if case["residual"] else 2) + (2 * rows * k if train else 0)
    else:
        vectors = k * ((2 if case["post"] else 0) + (2 if case["pre"] else 0) + (1 if case["gate"] == "channel" else 0))
        full = rows * k * (1 if case["gate"] == "full" else 0)
        count = rows * k * (4 if case["pre"] else 3) + vectors + full
        if train:
            count += rows * k * (4 if case["pre"] else 3) + vectors + full
    return {"bytes": float(count * e), "flops": _flops(case)}
