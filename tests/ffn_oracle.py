"""The feed-forward operators from their formulas in 64 bits: what tests/test_ffn_ops.py and tests/test_gpu_ffn.py compare with."""
import numpy as np
import torch

ACTS = {
    "none": lambda z: z,
    "relu": torch.relu,
    "silu": lambda z: z * torch.special.expit(z),
    "gelu": lambda z: z * torch.special.ndtr(z),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))),
    "sigmoid": torch.special.expit,
}


def linear(x, w, b=None, act="none", res=None):
    z = x @ w.T
    z = z if b is None else z + b
    y = ACTS[act](z)
    return y if res is None else y + res


def gated(x, wg, wu, bg=None, bu=None, act="silu"):
    return linear(x, wg, bg, act) * linear(x, wu, bu)


def norm(v, w, b, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    n = v / (v.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    return n if b is None else n + b


def residual_norm(x, y=None, kind="rms", eps=1e-6, pre_weight=None, pre_bias=None, post_weight=None, post_bias=None, gate=None,
                  scale=1.0):
    r = x
    if y is not None:
        n = y if post_weight is None else norm(y, post_weight, post_bias, kind, eps)
        r = x + scale * (n if gate is None else gate * n)
    return r, None if pre_weight is None else norm(r, pre_weight, pre_bias, kind, eps)


def philox4x32(counter, key, rounds):
    """One block: four 32-bit words, in Python integers."""
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(rounds):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ c3 ^ k1, a & 0xFFFFFFFF
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def kept(key, n, p):
    """Boolean numpy array: which of n elements stay."""
    seed, call = (int(v) & (2 ** 64 - 1) for v in key)
    words = []
    for e in range((n + 3) // 4):
        words += philox4x32((e & 0xFFFFFFFF, e >> 32, call & 0xFFFFFFFF, call >> 32), (seed & 0xFFFFFFFF, seed >> 32), 7)
    return np.array(words[:n], dtype=np.uint64) >= np.uint64(int(p * 2 ** 32))


def rounding(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2
