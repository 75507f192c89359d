"""Norms, gates and scales of residual blocks, as modules around ``ops.row_norm`` and ``ops.residual_norm``.

The reference's models stack their convolutions plainly (/root/reference/models/basicgnn_large.py:161-207), which stops
paying after a few layers; ``BasicGNN(residual=...)`` joins them through these modules instead."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.nn import Parameter

from .. import ops


class RowNorm(torch.nn.Module):
    """LayerNorm ("layer") or RMS norm ("rms", no bias) of every row."""

    def __init__(self, channels: int, kind: str = "layer", eps: float = 1e-5):
        super().__init__()
        if kind not in ("layer", "rms"):
            raise ValueError(f"kind is 'layer' or 'rms', got {kind!r}")
        self.kind, self.eps = kind, eps
        self.weight = Parameter(torch.empty(channels))
        self.register_parameter("bias", Parameter(torch.empty(channels)) if kind == "layer" else None)
        self.reset_parameters()

    def reset_parameters(self):
        torch.nn.init.ones_(self.weight)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, x: Tensor) -> Tensor:
        return ops.row_norm(x, self.weight, self.bias, self.kind, self.eps)

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}({self.weight.shape[0]}, {self.kind!r})"


class ResidualNorm(torch.nn.Module):
    """The join behind a block: ``out = x + scale * sigmoid(gate) * N_post(y)`` and ``h = N_pre(out)`` for the next block.

    post         norm of the block's output: "layer", "rms" or None
    pre          norm in front of the next block: "layer" or "rms"
    gate         None, "channel" (a learned vector), or "node" / "node_channel": a linear map of the block's input to one
                 gate per node, or per node and channel
    scale        factor of the branch; with ``learn_scale`` it starts a learned vector"""

    def __init__(self, channels: int, post: Optional[str] = "layer", pre: str = "layer", gate: Optional[str] = None, scale: float = 1.0,
                 learn_scale: bool = False, eps: float = 1e-5):
        super().__init__()
        if gate not in (None, "channel", "node", "node_channel"):
            raise ValueError(f"gate is None, 'channel', 'node' or 'node_channel', got {gate!r}")
        self.channels, self.gate_kind, self.initial_scale, self.eps = channels, gate, float(scale), eps
        self.post = RowNorm(channels, post, eps) if post is not None else None
        self.pre = RowNorm(channels, pre, eps)
        if learn_scale:
            self.scale = Parameter(torch.empty(channels))
        else:
            self.scale = self.initial_scale
        if gate == "channel":
            self.gate = Parameter(torch.empty(channels))
        elif gate is not None:
            self.gate = torch.nn.Linear(channels, 1 if gate == "node" else channels)
        self.reset_parameters()

    def reset_parameters(self):
        for norm in (self.post, self.pre):
            if norm is not None:
                norm.reset_parameters()
        if isinstance(self.scale, Parameter):
            torch.nn.init.constant_(self.scale, self.initial_scale)
        if self.gate_kind == "channel":
            torch.nn.init.zeros_(self.gate)
        elif self.gate_kind is not None:
            self.gate.reset_parameters()

    def forward(self, x: Tensor, y: Tensor, h: Tensor, normalise: bool = True):
        """``(out, next h)`` from the stream ``x``, the block's output ``y`` and the block's input ``h``; without ``normalise``
        only ``out``."""
        gate = None if self.gate_kind is None else self.gate if self.gate_kind == "channel" else self.gate(h)
        post, pre = self.post, self.pre
        kw = dict(pre=pre.kind, pre_weight=pre.weight, pre_bias=pre.bias) if normalise else {}
        if post is not None:
            kw.update(post=post.kind, post_weight=post.weight, post_bias=post.bias)
        return ops.residual_norm(x, y, gate=gate, gate_act=None if gate is None else "sigmoid", scale=self.scale, eps=self.eps, **kw)

    def __repr__(self) -> str:
        return (f"{self.__class__.__name__}({self.channels}, post={self.post.kind if self.post is not None else None!r}, "
                f"pre={self.pre.kind!r}, gate={self.gate_kind!r})")


__all__ = ["RowNorm", "ResidualNorm"]
