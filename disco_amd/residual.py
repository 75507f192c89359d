"""The join between two residual blocks, in one pass over the rows (``disco_residual_norm_forward`` / ``_backward``):

    out = x + scale * act(gate) * N_post(y)      y: what the block computed, x: the residual stream
    h   = N_pre(out)                             what the next block reads

and the norm before the first block (``row_norm``).  Both are differentiable in every tensor.  The reference normalises
hidden layers with stock BatchNorm (/root/reference/models/basicgnn_large.py:119-133) and has no residual blocks; deep
networks need them.  There is no CPU fallback.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_KINDS = {None: 0, "rms": 1, "layer": 2}
_ACTS = {None: 0, "sigmoid": 1, "tanh": 2}
_NO_GATE, _FULL, _ROW, _CHANNEL = 0, 1, 2, 3


class _Plan:
    """What a call does besides its tensors."""
    __slots__ = ("post", "pre", "gate", "act", "scale", "eps", "block_dtype", "param_dtype", "has_block")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy, with unit column stride and rows that do not overlap (a repeated row is left as it is)."""
    if t.shape[1] > 1 and t.stride(1) != 1 or 0 < t.stride(0) < t.shape[1] and t.shape[0] > 1 or t.stride(0) < 0:
        return t.contiguous()
    return t


def _empty(n: int, F: int, dtype, device) -> torch.Tensor:
    """float32 rows start on 16 bytes, as the propagation reads them best; others lie densely."""
    if dtype == torch.float32:
        return torch.empty((n, (F + 3) // 4 * 4), dtype=dtype, device=device)[:, :F]
    return torch.empty((n, F), dtype=dtype, device=device)


def _describe(plan, x, y, gate, scale, w1, b1, w2, b2) -> "_lib.ResidualNorm":
    p, types = _lib.ptr, _lib.DTYPES
    return _lib.ResidualNorm(
        x.shape[0], x.shape[1], x.stride(0), 0 if y is None else y.stride(0), gate.stride(0) if gate is not None else 0,
        p(x), p(y), p(gate), p(w1), p(b1), p(w2), p(b2), p(scale),
        types[x.dtype], types[plan.block_dtype], types[plan.param_dtype], int(plan.has_block), plan.post, plan.pre, plan.gate, plan.act,
        plan.scale, plan.eps)


def _forward(plan, x, y, gate, scale, w1, b1, w2, b2, keep: bool):
    n, F = x.shape
    device = x.device
    lib = _lib.load()
    with torch.cuda.device(device):
        out = _empty(n, F, x.dtype, device) if plan.has_block else None
        h = _empty(n, F, plan.block_dtype, device) if plan.pre else None
        stats = torch.empty(4 * n, dtype=torch.float32, device=device) if keep else None
        d = _describe(plan, x, y, gate, scale, w1, b1, w2, b2)
        _lib.check(lib.disco_residual_norm_forward(d, _lib.ptr(out), out.stride(0) if out is not None else 0, _lib.ptr(h),
                                                   h.stride(0) if h is not None else 0, _lib.ptr(stats), _lib.current_stream(device)),
                   "disco_residual_norm_forward")
    return out, h, stats


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, x, y, gate, scale, w1, b1, w2, b2):
        x = _rows(x)
        y = None if y is None else _rows(y)
        if plan.gate == _FULL:
            gate = _rows(gate)
        out, h, stats = _forward(plan, x, y, gate, scale, w1, b1, w2, b2, True)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, scale, w1, b1, w2, b2, stats)
        if out is None:
            return h
        return out if h is None else (out, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        plan = ctx.plan
        x, y, gate, scale, w1, b1, w2, b2, stats = ctx.saved_tensors
        dout, dh = (grads if len(grads) == 2 else (grads[0], None) if plan.has_block else (None, grads[0]))
        _, nx, ny, ng, ns, nw1, nb1, nw2, nb2 = ctx.needs_input_grad
        if dout is None and dh is None:
            return (None,) * 9
        n, F = x.shape
        device = x.device
        dout = None if dout is None else _rows(dout)
        dh = None if dh is None else _rows(dh)
        lib = _lib.load()
        with torch.cuda.device(device):
            def like(t, wanted):
                return torch.empty(t.shape, dtype=t.dtype, device=device) if wanted and t is not None else None

            # without a gradient of h the stream's gradient is that of out itself
            through = dh is None and dout is not None
            dx = dout if through and nx else like(x, nx)
            dy, dg, ds = like(y, ny), like(gate, ng), like(scale, ns)
            dw1, db1 = like(w1, nw1), like(b1, nb1)
            dw2, db2 = (like(w2, nw2), like(b2, nb2)) if dh is not None else (None, None)
            d = _describe(plan, x, y, gate, scale, w1, b1, w2, b2)
            nb = lib.disco_residual_norm_workspace_bytes(n, F)
            ws = torch.empty(max(int(nb), 1), dtype=torch.uint8, device=device)
            s0 = lambda t: t.stride(0) if t is not None else F  # noqa: E731
            p = _lib.ptr
            g = _lib.ResidualNormGrads(p(dout), p(dh), None if through else p(dx), p(dy), p(dg), s0(dout), s0(dh), s0(dx), s0(dy),
                                       s0(dg), p(dw1), p(db1), p(dw2), p(db2), p(ds))
            _lib.check(lib.disco_residual_norm_backward(d, p(stats), g, p(ws), ws.numel(), _lib.current_stream(device)),
                       "disco_residual_norm_backward")
        return None, dx, dy, dg, ds, dw1, db1, dw2, db2


def _check(t, what: str, shapes=None, device=None) -> None:
    if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
        raise TypeError(f"{what} must be a dense tensor")
    if shapes is not None and tuple(t.shape) not in shapes:
        raise ValueError(f"{what} must be of shape {' or '.join(str(list(s)) for s in shapes)}, got {list(t.shape)}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{what} is on {t.device}, x on {device}")


def _plan(x, block_dtype, post, pre, gate_kind, gate_act, scale, eps, has_block) -> _Plan:
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, width], got {list(x.shape)}")
    if not 1 <= x.shape[1] <= _lib.RESIDUAL_MAX_WIDTH:
        raise ValueError(f"width {x.shape[1]} is outside 1 .. {_lib.RESIDUAL_MAX_WIDTH}")
    if x.dtype not in _lib.DTYPES or block_dtype not in _lib.DTYPES or (x.dtype != block_dtype and x.dtype != torch.float32):
        raise TypeError(f"types are float32, float16 or bfloat16, the same for stream and block, or a float32 stream: got {x.dtype} and "
                        f"{block_dtype}")
    for kind in (post, pre):
        if kind not in _KINDS:
            raise ValueError(f"a norm is 'rms', 'layer' or None, got {kind!r}")
    if gate_act not in _ACTS:
        raise ValueError(f"gate_act is 'sigmoid', 'tanh' or None, got {gate_act!r}")
    if not (eps > 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be positive, got {eps}")
    plan = _Plan()
    plan.post, plan.pre, plan.gate, plan.act = _KINDS[post], _KINDS[pre], gate_kind, _ACTS[gate_act]
    plan.scale, plan.eps, plan.block_dtype, plan.has_block = float(scale), float(eps), block_dtype, has_block
    return plan


def _vectors(plan, x, vectors):
    """Parameter vectors on x's device, contiguous and of one type (mixed types meet in float32)."""
    dtypes = set()
    for name, v in vectors.items():
        if v is not None:
            _check(v, name, [(x.shape[1],)], x.device)
            if v.dtype not in _lib.DTYPES:
                raise TypeError(f"{name} must be float32, float16 or bfloat16, got {v.dtype}")
            dtypes.add(v.dtype)
    plan.param_dtype = dtypes.pop() if len(dtypes) == 1 else torch.float32
    return [None if v is None else v.to(plan.param_dtype).contiguous() for v in vectors.values()]


def _run(plan, *tensors):
    if tensors[0].device.type != "cuda":
        raise RuntimeError(f"x is on {tensors[0].device}: disco_amd runs on the GPU only, there is no CPU fallback")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _ResidualNormFn.apply(plan, *tensors)
    x, y, gate, *vectors = (None if t is None else t.detach() for t in tensors)
    out, h, _ = _forward(plan, _rows(x), None if y is None else _rows(y), _rows(gate) if plan.gate == _FULL else gate, *vectors, False)
    if out is None:
        return h
    return out if h is None else (out, h)


def row_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, kind: str = "layer",
             eps: float = 1e-5, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Normalised rows of ``x`` [rows, width]: the norm before the first block.

    kind   "layer": ``(x - mean) / sqrt(var + eps) * weight + bias``; "rms": ``x / sqrt(mean(x^2) + eps) * weight + bias``
    dtype  type of the result where it is not x's: a 16-bit block on a float32 stream."""
    _check(x, "x")
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'")
    plan = _plan(x, dtype or x.dtype, None, kind, _NO_GATE, None, 1.0, eps, False)
    weight, bias = _vectors(plan, x, {"weight": weight, "bias": bias})
    return _run(plan, x, None, None, None, None, None, weight, bias)


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, gate: Optional[torch.Tensor] = None, gate_act: Optional[str] = None,
                  scale: Union[float, torch.Tensor] = 1.0, post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out = x + scale * gate_act(gate) * N_post(y)``; with ``pre`` also ``h = N_pre(out)``, returned as ``(out, h)``.

    x, y       [rows, width]: the residual stream and the block's output.  Both float32, float16 or bfloat16, or a float32
               stream with a 16-bit block; ``out`` has x's type, ``h`` has y's.  ``h`` is the norm of the sum before it
               is rounded to x's type.
    gate       [rows, width] or [rows, 1] (y's type), or [width] (a parameter); ``gate_act`` is "sigmoid", "tanh" or None.
               With one row, [1, 1] is the row's gate (and so it is with a width of 1).
    scale      a number, or a vector [width] to be learned.
    post, pre  "rms", "layer" or None, each with an optional weight and bias [width] (float32 or 16-bit)."""
    _check(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, width], got {list(x.shape)}")
    n, F = x.shape
    _check(y, "y", [(n, F)], x.device)
    gate_kind, vector = _NO_GATE, None
    if gate is not None:
        _check(gate, "gate", [(n, F), (n, 1), (F,)], x.device)
        gate_kind = _CHANNEL if gate.dim() == 1 else _ROW if gate.shape[1] == 1 else _FULL
        if gate_kind != _CHANNEL and gate.dtype != y.dtype:
            raise TypeError(f"a gate for each row must be {y.dtype} like y, got {gate.dtype}")
    elif gate_act is not None:
        raise ValueError("gate_act needs a gate")
    if isinstance(scale, torch.Tensor):
        scale, vector = 1.0, scale
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if post is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need a post norm")
    if pre is None and (pre_weight is not None or pre_bias is not None):
        raise ValueError("pre_weight and pre_bias need a pre norm")
    plan = _plan(x, y.dtype, post, pre, gate_kind, gate_act, scale, eps, True)
    channel, vector, w1, b1, w2, b2 = _vectors(plan, x, {"gate": gate if gate_kind == _CHANNEL else None, "scale": vector,
                                                        "post_weight": post_weight, "post_bias": post_bias, "pre_weight": pre_weight,
                                                        "pre_bias": pre_bias})
    return _run(plan, x, y, channel if gate_kind == _CHANNEL else gate, vector, w1, b1, w2, b2)
