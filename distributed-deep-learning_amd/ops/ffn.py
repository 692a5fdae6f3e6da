"""Feed-forward operators: ``linear``, ``gated_linear``, ``dropout`` (+ ``DropoutRng``), ``residual_norm``.

Together they are the residual block of a model's trunk or head::

    h = gated_linear(n, w_gate, w_up, activation="silu")          # both projections, activation and product: one kernel
    y = linear(h, w_down, b_down)                                  # bias, activation and residual in the epilogue
    y = dropout(y, p, rng.next_key())                              # the mask is regenerated, never stored
    x, n = residual_norm(x, y, pre_weight=w, gate=g)               # join, and the next block's norm, in one pass

All four are differentiable once, by a backward pass (forward-mode tangents are refused on the GPU), take float32, bfloat16 and float16 (one type per call; the vectors of ``residual_norm`` may be
float32 beside 16-bit rows) and inputs of any strides, sum in fp32, and round a result once.  (16-bit gradients of products with
more than 32 rows read dz, the gradient in front of the activation, rounded to the type, as the matrix cores want it.)  On the GPU they run the kernels of
``csrc/ffn_*.hip`` on the current stream and can be captured into a graph; on the CPU the same functions are plain PyTorch.
Arguments that do not fit raise ``ValueError``; so do, on the GPU, more than 2^30 rows and products of more than 2^26 columns.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import require_ext

#: activations of ``linear`` and ``gated_linear``, in the order of csrc/ffn_common.h
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")
_ACT_ID = {a: i for i, a in enumerate(ACTIVATIONS)}
#: widest row of ``residual_norm``
MAX_NORM_WIDTH = 16384
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def act_id(activation: str) -> int:
    try:
        return _ACT_ID[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, got {activation!r}") from None


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _like(t: Optional[torch.Tensor], x: torch.Tensor, name: str, shape=None) -> None:
    if t is not None:
        _need(t.device == x.device and t.dtype == x.dtype, f"{name}: {t.dtype} on {t.device} beside {x.dtype} on {x.device}")
        _need(shape is None or tuple(t.shape) == tuple(shape), f"{name}: {tuple(shape or ())} expected, got {tuple(t.shape)}")


def _act(z: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "relu":
        return torch.relu(z)
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        c = z.clamp(-12, 12)                     # beyond, the sigmoid is 0 or 1 in fp32, and the cube would overflow in its derivative
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (c + 0.044715 * c ** 3))
    return torch.sigmoid(z) if activation == "sigmoid" else z


def _project(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], names: Tuple[str, str]) -> torch.Tensor:
    """x w^T + b in fp32 (CPU path)."""
    _need(x.dtype in _TYPES, f"x: float32, bfloat16 or float16 expected, got {x.dtype}")
    _need(x.dim() >= 1 and w.dim() == 2 and x.shape[-1] == w.shape[1],
          f"x [.., K] and {names[0]} [N, K] expected, got {tuple(x.shape)} and {tuple(w.shape)}")
    _like(w, x, names[0])
    _like(b, x, names[1], (w.shape[0],))
    z = x.float() @ w.float().t()
    return z if b is None else z + b.float()


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: x [.., K], weight [N, K], bias [N], residual [.., N].

    Bias, activation and residual are the product's epilogue.  Training keeps x, weight and - with an activation - the fp32
    sums in front of it, so that the activation's slope is taken from unrounded sums.  On the GPU an operand that the kernels cannot
    read in place (a width off 16 bytes, strides) is kept as the copy they read: a second copy of such a weight until ``backward``,
    and the gradients are those of the values at the call even if the tensor is changed in place between."""
    a = act_id(activation)
    if x.is_cuda:
        return require_ext().linear(x, weight, bias, residual, a)
    y = _act(_project(x, weight, bias, ("weight", "bias")), activation)
    _like(residual, x, "residual", y.shape)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                 b_up: Optional[torch.Tensor] = None, activation: str = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)``: x [.., K], weights [F, K], both biases [F] or none.

    Both projections are one kernel; neither is written to memory at inference.  Training keeps both in fp32, and x and the weights
    as ``linear`` does."""
    a = act_id(activation)
    if x.is_cuda:
        return require_ext().gated_linear(x, w_gate, w_up, b_gate, b_up, a)
    _need(w_gate.shape == w_up.shape, f"w_gate {tuple(w_gate.shape)} and w_up {tuple(w_up.shape)} differ")
    _need((b_gate is None) == (b_up is None), "both biases or none")
    g, u = _project(x, w_gate, b_gate, ("w_gate", "b_gate")), _project(x, w_up, b_up, ("w_up", "b_up"))
    return (_act(g, activation) * u).to(x.dtype)


# --------------------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------------------
class DropoutRng:
    """Keys for ``dropout``: ``seed`` and a call counter that lives on the device.

    ``next_key()`` takes the next key with one small launch; captured into a graph, every replay takes a new one.  The counter
    advances atomically, so two streams never get the same key (which of them gets which is not defined: give each its own
    ``stream``).  ``stream`` selects one of 2**15 disjoint ranges of 2**48 calls."""

    def __init__(self, seed: int, device, stream: int = 0) -> None:
        _need(0 <= stream < 2 ** 15, f"stream must lie in [0, 2**15), got {stream}")
        seed = int(seed) % 2 ** 64
        seed = seed - 2 ** 64 if seed >= 2 ** 63 else seed          # the same 64 bits as a signed number
        self.stream = stream
        self.state = torch.tensor([seed, stream << 48], dtype=torch.int64, device=device)

    def seek(self, call: int) -> None:
        """The next key is call number ``call`` (0 <= call < 2**48) of this generator's stream: a resumed program goes on where it was.
        (Between captured steps, not in one: every replay would seek again.)"""
        _need(0 <= call < 2 ** 48, f"call must lie in [0, 2**48), got {call}")
        self.state[1].fill_((self.stream << 48) + call)

    def keys(self, n: int) -> torch.Tensor:
        """The next ``n`` keys, [n, 2]."""
        if self.state.is_cuda:
            return require_ext().rng_keys(self.state, n)
        _need(n >= 1, f"at least one key, got {n}")
        keys = self.state.repeat(n, 1)
        keys[:, 1] += torch.arange(n)
        self.state[1] += n
        return keys

    def next_key(self) -> torch.Tensor:
        return self.keys(1)[0]


def _kept(key: torch.Tensor, n: int, p: float) -> torch.Tensor:
    """Which of n elements a call keeps (CPU path): word e % 4 of Philox4x32-7 at (e // 4, call) under ``seed``, >= p * 2**32."""
    m = 0xFFFFFFFF
    e = torch.arange((n + 3) // 4, dtype=torch.int64)
    seed, call = int(key[0]), int(key[1])
    c = [e & m, e >> 32, torch.full_like(e, call & m), torch.full_like(e, (call >> 32) & m)]
    k = [seed & m, (seed >> 32) & m]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57                  # wraps; the low 64 bits are the product
        c = [((b >> 32) & m) ^ c[1] ^ k[0], b & m, ((a >> 32) & m) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return torch.stack(c, 1).reshape(-1)[:n] >= int(p * 2 ** 32)


def dropout(x: torch.Tensor, p: float, key: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + keep * x / (1 - p)``; each element of x is dropped with probability ``p`` (0 <= p <= 1).

    ``key`` is two int64 values on x's device (``DropoutRng.next_key()``): the same key drops the same elements, whatever the
    type and strides of x, and the backward pass draws them again instead of reading a mask.  A dropped element contributes
    zero even if it is infinite or NaN."""
    if x.is_cuda:
        return require_ext().dropout(x, p, key, residual)
    _need(x.dtype in _TYPES, f"x: float32, bfloat16 or float16 expected, got {x.dtype}")
    _need(0 <= p <= 1, f"p must lie in [0, 1], got {p}")
    _need(key.dtype == torch.int64 and key.numel() == 2 and key.device == x.device,
          "key must be two int64 values (seed, call) on the input's device")
    _like(residual, x, "residual", x.shape)
    keep = _kept(key.reshape(2), x.numel(), p).reshape(x.shape)
    y = torch.where(keep, x.float() * (1 / (1 - p) if p < 1 else 0.0), 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


# --------------------------------------------------------------------------------------
# residual join with the norms on both sides
# --------------------------------------------------------------------------------------
def _norm(v: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], kind: str, eps: float) -> torch.Tensor:
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.float()
    return n if b is None else n + b.float()


def residual_norm(x: torch.Tensor, branch: Optional[torch.Tensor] = None, kind: str = "rms", eps: float = 1e-6,
                  pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None,
                  scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``r = x + scale * gate * post(branch)``, ``h = pre(r)``; returns ``(r, h)``.

    ``post`` is the norm behind the finished block (there if ``post_weight`` is given), ``pre`` the one in front of the next (there
    if ``pre_weight`` is given; else h is None).  ``kind``: ``"layer"`` (mean and variance, optional biases) or ``"rms"`` (no
    biases).  ``gate`` is one value per channel [C] or a tensor of x's shape.  Without a branch r is x itself: a plain norm.
    Rows have 1 to 16384 columns.  h is taken from the unrounded r."""
    _need(kind in ("rms", "layer"), f"kind must be 'rms' or 'layer', got {kind!r}")
    if x.is_cuda:
        return require_ext().residual_norm(x, branch, gate, post_weight, post_bias, pre_weight, pre_bias, kind == "layer", eps,
                                           scale)
    _need(x.dtype in _TYPES, f"x: float32, bfloat16 or float16 expected, got {x.dtype}")
    _need(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_NORM_WIDTH, f"x [.., C] with 1 <= C <= {MAX_NORM_WIDTH} expected, got {tuple(x.shape)}")
    _need(eps >= 0, "eps must not be negative")
    _need(kind == "layer" or (post_bias is None and pre_bias is None), "an RMS norm has no bias")
    _need(post_weight is not None or post_bias is None, "post_bias without post_weight")
    _need(pre_weight is not None or pre_bias is None, "pre_bias without pre_weight")
    _need(branch is not None or (gate is None and post_weight is None), "gate or post_weight without a branch")
    _need(branch is not None or pre_weight is not None, "neither a branch nor pre_weight: nothing to do")
    _like(branch, x, "branch", x.shape)
    full = gate is not None and (gate.dim() != 1 or (x.dim() == 1 and gate.dtype == x.dtype))
    vectors = [v for v in (post_weight, post_bias, pre_weight, pre_bias, None if full else gate) if v is not None]
    for v in vectors:
        _need(tuple(v.shape) == (x.shape[-1],) and v.device == x.device, f"a vector [{x.shape[-1]}] expected, got {tuple(v.shape)}")
        _need(v.dtype in (x.dtype, torch.float32) and v.dtype == vectors[0].dtype,
              f"weights, biases and a channel gate share one type, float32 or {x.dtype}")
    if full:
        _like(gate, x, "gate", x.shape)
    r = x.float()
    if branch is not None:
        n = branch.float() if post_weight is None else _norm(branch.float(), post_weight, post_bias, kind, eps)
        r = r + scale * (n if gate is None else gate.float() * n)
    h = None if pre_weight is None else _norm(r, pre_weight, pre_bias, kind, eps).to(x.dtype)
    return (x if branch is None else r.to(x.dtype)), h
