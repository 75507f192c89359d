"""The join between two residual blocks, in one pass over the rows (``disco_residual_norm_forward`` / ``_backward``):

    out = x + scale * act(gate) * N_post(y)      y: what the block computed, x: the residual stream
    h   = N_pre(out)                             what the next block reads

and the norm before the first block (``row_norm``).  Both are differentiable in every tensor.  The reference normalises
hidden layers with stock BatchNorm (/root/reference/models/basicgnn_large.py:119-133) and has no residual blocks; deep
networks need them.  There is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_KINDS = {None: 0, "rms": 1, "layer": 2}
_ACTS = {None: 0, "sigmoid": 1, "tanh": 2}
_NO_GATE, _FULL, _ROW, _CHANNEL = 0, 1, 2, 3
_DTYPES = _lib.DTYPES
_F32 = torch.float32
_LEAST, _MOST = torch.finfo(_F32).tiny, torch.finfo(_F32).max


class _Plan:
    """What a call does besides its tensors."""
    __slots__ = ("post", "pre", "gate", "act", "scale", "eps", "block_dtype", "param_dtype", "has_block", "index")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy, with unit column stride and rows that do not overlap (a repeated row is left as it is)."""
    if t.is_contiguous():
        return t
    n, F = t.shape
    r, c = t.stride()
    if F > 1 and c != 1 or n > 1 and 0 < r < F:
        return t.contiguous()
    return t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _describe(plan, x, y, gate, scale, w1, b1, w2, b2) -> "_lib.ResidualNorm":
    n, F = x.shape
    return _lib.ResidualNorm(
        n, F, x.stride(0), 0 if y is None else y.stride(0), 0 if gate is None else gate.stride(0), x.data_ptr(), _ptr(y), _ptr(gate),
        _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2), _ptr(scale), _DTYPES[x.dtype], _DTYPES[plan.block_dtype], _DTYPES[plan.param_dtype],
        plan.has_block, plan.post, plan.pre, plan.gate, plan.act, plan.scale, plan.eps)


def _forward(plan, x, y, gate, scale, w1, b1, w2, b2, keep: bool):
    if plan.index != torch.cuda.current_device():
        with torch.cuda.device(plan.index):
            return _forward(plan, x, y, gate, scale, w1, b1, w2, b2, keep)
    # dense rows: columns that nothing writes between them leave cache lines half written (the norm of 2.4 M rows of 41 floats:
    # 268 us with rows padded to 44, 170 dense)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if plan.has_block else None
    h = torch.empty(x.shape, dtype=plan.block_dtype, device=x.device) if plan.pre else None
    stats = torch.empty(4 * x.shape[0], dtype=_F32, device=x.device) if keep else None
    status = _lib.load().disco_residual_norm_forward(
        _describe(plan, x, y, gate, scale, w1, b1, w2, b2), _ptr(out), 0 if out is None else out.stride(0), _ptr(h),
        0 if h is None else h.stride(0), _ptr(stats), _lib.stream_of(plan.index))
    if status:
        _lib.check(status, "disco_residual_norm_forward")
    return out, h, stats


def _backward(plan, needs, dout, dh, x, y, gate, scale, w1, b1, w2, b2, stats):
    if plan.index != torch.cuda.current_device():
        with torch.cuda.device(plan.index):
            return _backward(plan, needs, dout, dh, x, y, gate, scale, w1, b1, w2, b2, stats)
    n, F = x.shape
    dout = None if dout is None else _rows(dout)
    dh = None if dh is None else _rows(dh)

    def like(t, wanted):
        return torch.empty(t.shape, dtype=t.dtype, device=t.device) if wanted and t is not None else None

    nx, ny, ng, ns, nw1, nb1, nw2, nb2 = needs
    # without a gradient of h the stream's gradient is that of out itself
    through = dh is None
    dx = (dout if nx else None) if through else like(x, nx)
    dy, dg, ds, dw1, db1 = like(y, ny), like(gate, ng), like(scale, ns), like(w1, nw1), like(b1, nb1)
    dw2, db2 = (None, None) if through else (like(w2, nw2), like(b2, nb2))
    lib = _lib.load()
    nb = lib.disco_residual_norm_workspace_bytes(n, F)
    ws = torch.empty(nb, dtype=torch.uint8, device=x.device)

    def stride(t):
        return F if t is None else t.stride(0)

    g = _lib.ResidualNormGrads(_ptr(dout), _ptr(dh), 0 if through else _ptr(dx), _ptr(dy), _ptr(dg), stride(dout), stride(dh), stride(dx),
                               stride(dy), stride(dg), _ptr(dw1), _ptr(db1), _ptr(dw2), _ptr(db2), _ptr(ds))
    status = lib.disco_residual_norm_backward(_describe(plan, x, y, gate, scale, w1, b1, w2, b2), _ptr(stats), g, ws.data_ptr(), nb,
                                              _lib.stream_of(plan.index))
    if status:
        _lib.check(status, "disco_residual_norm_backward")
    return None, dx, dy, dg, ds, dw1, db1, dw2, db2


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, x, y, gate, scale, w1, b1, w2, b2):
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
        dout, dh = grads if len(grads) == 2 else (grads[0], None) if plan.has_block else (None, grads[0])
        if dout is None and dh is None:
            return (None,) * 9
        return _backward(plan, ctx.needs_input_grad[1:], dout, dh, *ctx.saved_tensors)


def _matrix(x, what: str):
    if not isinstance(x, torch.Tensor) or x.layout is not torch.strided:
        raise TypeError(f"{what} must be a dense tensor")
    if x.dim() != 2:
        raise ValueError(f"{what} must be [rows, width], got {list(x.shape)}")
    return x


def _plan(x, block_dtype, post, pre, gate_kind, gate_act, scale, eps, has_block, vectors) -> _Plan:
    """Checks what the tensors and options have to be, and settles the parameters' type: theirs, or float32 where they differ."""
    F, device = x.shape[1], x.device
    if not 1 <= F <= _lib.RESIDUAL_MAX_WIDTH:
        raise ValueError(f"width {F} is outside 1 .. {_lib.RESIDUAL_MAX_WIDTH}")
    if x.dtype not in _DTYPES or block_dtype not in _DTYPES or (x.dtype != block_dtype and x.dtype != _F32):
        raise TypeError(f"types are float32, float16 or bfloat16, the same for stream and block, or a float32 stream: got {x.dtype} and "
                        f"{block_dtype}")
    if post not in _KINDS or pre not in _KINDS:
        raise ValueError(f"a norm is 'rms', 'layer' or None, got {post!r} and {pre!r}")
    if gate_act not in _ACTS:
        raise ValueError(f"gate_act is 'sigmoid', 'tanh' or None, got {gate_act!r}")
    if not _LEAST <= eps <= _MOST:
        raise ValueError(f"eps must be positive and finite in float32, got {eps}")
    dtype = None
    for name, v in vectors:
        if v is None:
            continue
        if not isinstance(v, torch.Tensor) or v.layout is not torch.strided:
            raise TypeError(f"{name} must be a dense tensor")
        if v.shape != (F,):
            raise ValueError(f"{name} must be of shape [{F}], got {list(v.shape)}")
        if v.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float32, float16 or bfloat16, got {v.dtype}")
        if v.device != device:
            raise RuntimeError(f"{name} is on {v.device}, x on {device}")
        dtype = v.dtype if dtype is None or dtype == v.dtype else _F32
    if not x.is_cuda:
        raise RuntimeError(f"x is on {device}: disco_amd runs on the GPU only, there is no CPU fallback")
    plan = _Plan()
    plan.post, plan.pre, plan.gate, plan.act = _KINDS[post], _KINDS[pre], gate_kind, _ACTS[gate_act]
    plan.scale, plan.eps, plan.block_dtype, plan.has_block = scale, eps, block_dtype, has_block
    plan.param_dtype, plan.index = dtype or _F32, x.get_device()
    return plan


def _run(plan, x, y, gate, vectors):
    """The call itself: tensors as the kernels read them, through autograd where one of them needs a gradient."""
    x = _rows(x)
    if y is not None:
        y = _rows(y)
    if plan.gate == _FULL:
        gate = _rows(gate)
    grads = torch.is_grad_enabled() and (x.requires_grad or (y is not None and y.requires_grad) or (gate is not None and gate.requires_grad))
    dtype = plan.param_dtype
    tensors = [x, y, gate]
    for name, v in vectors:
        if v is not None:
            grads = grads or (v.requires_grad and torch.is_grad_enabled())
            if v.dtype != dtype:
                v = v.to(dtype)
            if not v.is_contiguous():
                v = v.contiguous()
        if name == "gate":
            if v is not None:
                tensors[2] = v
        else:
            tensors.append(v)
    if grads:
        return _ResidualNormFn.apply(plan, *tensors)
    out, h, _ = _forward(plan, *tensors, False)
    if out is None:
        return h
    return out if h is None else (out, h)


def row_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, kind: str = "layer",
             eps: float = 1e-5, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Normalised rows of ``x`` [rows, width]: the norm before the first block.

    kind   "layer": ``(x - mean) / sqrt(var + eps) * weight + bias``; "rms": ``x / sqrt(mean(x^2) + eps) * weight + bias``
    dtype  type of the result where it is not x's: a 16-bit block on a float32 stream."""
    _matrix(x, "x")
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'")
    vectors = (("scale", None), ("post_weight", None), ("post_bias", None), ("weight", weight), ("bias", bias))
    return _run(_plan(x, dtype or x.dtype, None, kind, _NO_GATE, None, 1.0, eps, False, vectors), x, None, None, vectors)


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, gate: Optional[torch.Tensor] = None, gate_act: Optional[str] = None,
                  scale: Union[float, torch.Tensor] = 1.0, post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out = x + scale * gate_act(gate) * N_post(y)``; with ``pre`` also ``h = N_pre(out)``, returned as ``(out, h)``.

    x, y       [rows, width]: the residual stream and the block's output.  Both float32, float16 or bfloat16, or a float32
               stream with a 16-bit block; ``out`` has x's type, ``h`` has y's.  ``h`` is the norm of the sum before it
               is rounded to x's type.
    gate       [rows, width] or [rows, 1] (y's type), or [width] (a parameter); ``gate_act`` is "sigmoid", "tanh" or None.
    scale      a number, or a vector [width] to be learned.
    post, pre  "rms", "layer" or None, each with an optional weight and bias [width] (float32 or 16-bit)."""
    _matrix(x, "x")
    _matrix(y, "y")
    if y.shape != x.shape:
        raise ValueError(f"y must be of x's shape {list(x.shape)}, got {list(y.shape)}")
    if y.device != x.device:
        raise RuntimeError(f"y is on {y.device}, x on {x.device}")
    kind, vector, channel = _NO_GATE, None, None
    if gate is not None:
        if isinstance(gate, torch.Tensor) and gate.dim() == 1:
            kind, channel, gate = _CHANNEL, gate, None
        else:
            _matrix(gate, "gate")
            n, F = x.shape
            if gate.shape != (n, F) and gate.shape != (n, 1):
                raise ValueError(f"gate must be of shape [{n}, {F}], [{n}, 1] or [{F}], got {list(gate.shape)}")
            if gate.dtype != y.dtype:
                raise TypeError(f"a gate for each row must be {y.dtype} like y, got {gate.dtype}")
            if gate.device != x.device:
                raise RuntimeError(f"gate is on {gate.device}, x on {x.device}")
            kind = _ROW if gate.shape[1] == 1 else _FULL
    elif gate_act is not None:
        raise ValueError("gate_act needs a gate")
    if isinstance(scale, torch.Tensor):
        scale, vector = 1.0, scale
    elif not -_MOST <= scale <= _MOST:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    if post is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need a post norm")
    if pre is None and (pre_weight is not None or pre_bias is not None):
        raise ValueError("pre_weight and pre_bias need a pre norm")
    vectors = (("gate", channel), ("scale", vector), ("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight),
               ("pre_bias", pre_bias))
    return _run(_plan(x, y.dtype, post, pre, kind, gate_act, scale, eps, True, vectors), x, y, gate, vectors)
