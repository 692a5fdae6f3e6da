"""Classifier heads between the pooled features and the class logits.

``linear`` is the reference's head, one ``Linear(1024, classes)`` (single.py:299).  ``gated`` puts a residual feed-forward block
in front of it::

    h = layer_norm(f)
    y = dropout(W_down (silu(W_gate h + b_gate) * (W_up h + b_up)) + b_down)
    logits = classifier(layer_norm(f + scale * y))            # ``scale``: one learned value per channel, 0.1 at the start

for fine-tuning on frozen or slowly trained features.  The native engine computes it in fp32 under every ``--dtype``, like the
linear classifier.  The block's parameters live under ``ffn.`` in the state-dict; everything
else keeps its name, so checkpoints of either head load into the other's backbone.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Tuple

import torch
import torch.nn as nn

from .. import ops

HEADS = ("linear", "gated")


@dataclass(frozen=True)
class HeadConfig:
    """``width``: hidden columns of the gated block; ``dropout``: probability on its output in training."""
    kind: str = "linear"
    width: int = 1024
    dropout: float = 0.1

    def __post_init__(self) -> None:
        if self.kind not in HEADS:
            raise ValueError(f"head must be one of {HEADS}, got {self.kind!r}")
        if self.width < 1:
            raise ValueError(f"head width must be positive, got {self.width}")
        if not 0.0 <= self.dropout < 1.0:
            raise ValueError(f"head dropout must lie in [0, 1), got {self.dropout}")


def dropout_seed() -> int:
    """The process's seed (``--seed``, or what torch drew), another one on every rank."""
    rank = torch.distributed.get_rank() if torch.distributed.is_available() and torch.distributed.is_initialized() else 0
    return (torch.initial_seed() + 0x9E3779B97F4A7C15 * rank) % 2 ** 64


def first_call(epoch: int) -> int:
    """Where an epoch's dropout keys start: like the order of the data, the masks follow from the seed and the epoch, so a run that is
    resumed at an epoch draws what the uninterrupted one drew."""
    return (epoch % 2 ** 16) << 32


class GatedHead(nn.Module):
    """The block in front of the classifier; ``forward`` is the portable path."""

    def __init__(self, channels: int, cfg: HeadConfig) -> None:
        super().__init__()
        self.dropout = cfg.dropout
        self.norm_in = nn.LayerNorm(channels)
        self.gate = nn.Linear(channels, cfg.width)
        self.up = nn.Linear(channels, cfg.width)
        self.down = nn.Linear(cfg.width, channels)
        self.scale = nn.Parameter(torch.full((channels,), 0.1))
        self.norm_out = nn.LayerNorm(channels)
        self._rng: Optional[ops.DropoutRng] = None
        self._epoch = 0

    def set_epoch(self, epoch: int) -> None:
        self._epoch = epoch
        if self._rng is not None:
            self._rng.seek(first_call(epoch))

    def rng(self, device) -> ops.DropoutRng:
        """The keys' generator on ``device``; it goes where the features go, and on with its sequence."""
        if self._rng is None:
            self._rng = ops.DropoutRng(dropout_seed(), device)
            self._rng.seek(first_call(self._epoch))
        elif self._rng.state.device != torch.device(device):
            self._rng.state = self._rng.state.to(device)
        return self._rng

    def forward(self, f: torch.Tensor) -> torch.Tensor:
        _, h = ops.residual_norm(f, kind="layer", eps=self.norm_in.eps, pre_weight=self.norm_in.weight, pre_bias=self.norm_in.bias)
        y = ops.gated_linear(h, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, activation="silu")
        y = ops.linear(y, self.down.weight, self.down.bias)
        if self.training and self.dropout > 0:
            y = ops.dropout(y, self.dropout, self.rng(f.device).next_key())
        return ops.residual_norm(f, y, kind="layer", eps=self.norm_out.eps, gate=self.scale, pre_weight=self.norm_out.weight,
                                 pre_bias=self.norm_out.bias)[1]


#: parameters of the block in the order the native head binds them
PARAMS = ("norm_in.weight", "norm_in.bias", "gate.weight", "up.weight", "gate.bias", "up.bias", "down.weight", "down.bias", "scale",
          "norm_out.weight", "norm_out.bias")
LAYER_NORM_EPS = 1e-5


def native_forward(ext, p: Dict[str, torch.Tensor], f: torch.Tensor, drop: float, key: Optional[torch.Tensor],
                   keep: bool) -> Tuple[torch.Tensor, Tuple[Optional[torch.Tensor], ...]]:
    """The block on the parameter views of the native engine: (h, what the backward pass needs).  ``key`` None: no dropout.  ``keep``:
    a backward pass may follow; otherwise neither the projections' sums nor the norms' statistics are written."""
    silu = ops.ACTIVATIONS.index("silu")
    _, n, s_in = ext.norm_forward(f, None, None, None, None, p["norm_in.weight"], p["norm_in.bias"], True, LAYER_NORM_EPS, 1.0, keep)
    g, z = ext.gated_forward(n, p["gate.weight"], p["up.weight"], p["gate.bias"], p["up.bias"], silu, keep)
    y, _ = ext.linear_forward(g, p["down.weight"], p["down.bias"], None, 0, False)
    if key is not None:
        y = ext.dropout(y, drop, key, None)
    _, h, s_out = ext.norm_forward(f, y, p["scale"], None, None, p["norm_out.weight"], p["norm_out.bias"], True, LAYER_NORM_EPS, 1.0,
                                   keep)
    return h, (f, n, s_in, z, g, y, s_out)


def native_backward(ext, p: Dict[str, torch.Tensor], saved, drop: float, key: Optional[torch.Tensor],
                    dh: torch.Tensor) -> Tuple[torch.Tensor, List[torch.Tensor]]:
    """(gradient of the features, gradients of ``PARAMS``)"""
    silu = ops.ACTIVATIONS.index("silu")
    f, n, s_in, z, g, y, s_out = saved
    df, dy, dscale, _, _, dw_out, db_out = ext.norm_backward(f, y, p["scale"], None, None, p["norm_out.weight"], p["norm_out.bias"], True,
                                                             LAYER_NORM_EPS, 1.0, s_out, None, dh)
    if key is not None:
        dy = ext.dropout(dy, drop, key, None)
    dg, dw_down, db_down = ext.linear_backward(dy, g, p["down.weight"], None, 0, True, True, True)
    dn, dw_gate, dw_up, db_gate, db_up = ext.gated_backward(dg, n, p["gate.weight"], p["up.weight"], z, silu, True, True, True)
    df_in, _, _, _, _, dw_in, db_in = ext.norm_backward(f, None, None, None, None, p["norm_in.weight"], p["norm_in.bias"], True,
                                                        LAYER_NORM_EPS, 1.0, s_in, None, dn)
    return df.add_(df_in), [dw_in, db_in, dw_gate, dw_up, db_gate, db_up, dw_down, db_down, dscale, dw_out, db_out]
