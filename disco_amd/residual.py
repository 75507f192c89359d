"""The join between two residual blocks, in one pass over the rows (``disco_residual_norm_forward`` / ``_backward``):

    out = x + scale * act(gate) * N_post(y)      y: what the block computed, x: the residual stream
    h   = N_pre(out)                             what the next block reads

and the norm before the first block (``row_norm``).  Both are differentiable in every tensor.  The reference normalises
hidden layers with stock BatchNorm (/root/reference/models/basicgnn_large.py:119-133) and has no residual blocks; deep
networks need them.  The arguments are checked here; the autograd node is disco_torch.cpp's.  Sums of squares are float32: entries
up to about 1e17.  Second and forward-mode derivatives are refused.  There is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from . import _lib

_KINDS = {None: 0, "rms": 1, "layer": 2}
_ACTS = {None: 0, "sigmoid": 1, "tanh": 2}
_NO_GATE, _FULL, _ROW, _CHANNEL = 0, 1, 2, 3
_DTYPES = _lib.DTYPES
_F32 = torch.float32
_LEAST, _MOST = torch.finfo(_F32).tiny, torch.finfo(_F32).max


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy, with unit column stride and rows that do not overlap (a repeated row is left as it is)."""
    if t.is_contiguous():
        return t
    n, F = t.shape
    r, c = t.stride()
    if F > 1 and c != 1 or n > 1 and 0 < r < F:
        return t.contiguous()
    return t


def _matrix(x, what: str):
    if not isinstance(x, torch.Tensor) or x.layout is not torch.strided:
        raise TypeError(f"{what} must be a dense tensor")
    if x.dim() != 2:
        raise ValueError(f"{what} must be [rows, width], got {list(x.shape)}")
    return x


def _plan(x, block_dtype, post, pre, gate_kind, gate_act, eps, has_block, vectors):
    """Checks what the tensors and options have to be.  Returns the call's options, packed as disco_torch.cpp reads them, and the
    parameters' type: theirs, or float32 where they differ."""
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
    dtype = dtype or _F32
    return (_KINDS[post] | _KINDS[pre] << 2 | gate_kind << 4 | _ACTS[gate_act] << 6 | _DTYPES[block_dtype] << 8 | _DTYPES[dtype] << 10
            | has_block << 12), dtype


def _vector(v, dtype):
    if v is None:
        return None
    if v.dtype != dtype:
        v = v.to(dtype)
    return v if v.is_contiguous() else v.contiguous()


def _run(plan, x, y, gate, scale, eps, vectors):
    """The call itself, of tensors as the kernels read them; through autograd where one of them needs a gradient."""
    options, dtype = plan
    (_, channel), *rest = vectors
    if channel is not None:
        gate = _vector(channel, dtype)
    elif gate is not None and gate.shape[1] > 1:
        gate = _rows(gate)
    return _lib.torch_op("residual_norm")(_rows(x), None if y is None else _rows(y), gate, *[_vector(v, dtype) for _, v in rest], options, scale, eps)


def row_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, kind: str = "layer",
             eps: float = 1e-5, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Normalised rows of ``x`` [rows, width]: the norm before the first block.

    kind   "layer": ``(x - mean) / sqrt(var + eps) * weight + bias``; "rms": ``x / sqrt(mean(x^2) + eps) * weight + bias``
    dtype  type of the result where it is not x's: a 16-bit block on a float32 stream."""
    _matrix(x, "x")
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'")
    vectors = (("gate", None), ("scale", None), ("post_weight", None), ("post_bias", None), ("weight", weight), ("bias", bias))
    return _run(_plan(x, dtype or x.dtype, None, kind, _NO_GATE, None, eps, False, vectors), x, None, None, 1.0, eps, vectors)[0]


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
    got = _run(_plan(x, y.dtype, post, pre, kind, gate_act, eps, True, vectors), x, y, gate, scale, eps, vectors)
    return got[0] if pre is None else tuple(got)
