"""The norm over all gradients of a model, and clipping (``disco_grad_norm`` / ``disco_grad_clip``).

Any number of tensors, float32 / float16 / bfloat16 in any mixture, in two or three launches; the norm stays on the device,
nothing synchronises.  No counterpart in the reference, whose training loops do not clip
(/root/reference/LargeScaleCondensing.py:187-200).  There is no CPU fallback.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib

_NORMS = {1.0: 1, 2.0: 2, math.inf: 0}
_SHARED = "clip_grads: two tensors share memory; each gradient may be scaled only once"


def _list(tensors) -> List[torch.Tensor]:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not all([isinstance(t, torch.Tensor) for t in tensors]):
        raise TypeError("gradients must be dense tensors")
    return tensors


def _check(grads, out=()) -> None:
    """Says what is wrong with tensors that the kernels did not take, if it is not how they lie."""
    for g in [*grads, *out]:
        if g.layout is not torch.strided:
            raise TypeError("gradients must be dense tensors")
        if g.dtype not in _lib.DTYPES:
            raise TypeError(f"gradients must be float32, float16 or bfloat16, got {g.dtype}")
    for g, o in zip(grads, out):
        if o.shape != g.shape or o.device != g.device or o.dtype not in (g.dtype, torch.float32):
            raise ValueError(f"out must have the gradients' shapes and device and their type or float32, got {tuple(o.shape)} "
                             f"{o.dtype} on {o.device} for {tuple(g.shape)} {g.dtype} on {g.device}")
    for g in grads:
        if g.device != grads[0].device:
            raise ValueError(f"gradients on {grads[0].device} and {g.device}: one device at a time")
    if not grads[0].is_cuda:
        raise RuntimeError(f"gradients on {grads[0].device}: disco_amd runs on the GPU only, there is no CPU fallback")


def _norm_type(norm_type) -> int:
    p = _NORMS.get(float(norm_type))
    if p is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type!r}")
    return p


def _launch(grads: Sequence[torch.Tensor], out, p: int, max_norm: float) -> Optional[torch.Tensor]:
    """The norm, and the clipping into ``out`` where that is given; None where the kernels do not read the tensors as they are."""
    return _lib.torch_op("gradient_norm")(grads, out, p, max_norm)


def grad_norm(grads: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """``(sum |g|^p)^(1/p)`` over every element of every tensor, p = ``norm_type`` in {1, 2, inf}; a float32 scalar on the
    device.  Sums run in float64 in a fixed order: nothing overflows in between (a norm beyond float32 is infinite), and the
    result does not vary.  It has no derivative: where a gradient requires one itself, differentiating the norm raises."""
    p = _norm_type(norm_type)
    grads = _list(grads)
    if not grads:
        return torch.zeros((), dtype=torch.float32, device="cuda" if torch.cuda.is_available() else "cpu")
    norm = _launch(grads, None, p, 0.0)
    if norm is None:
        _check(grads)
        norm = _launch([g.contiguous() for g in grads], None, p, 0.0)
    return norm


def clip_grads(grads: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales every gradient by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm before (float32, on the device).

    In place by default; ``out`` names one destination per gradient, of its shape and either its type or float32 (the
    buffers a mixed-precision optimiser reads).  Destinations that share memory are refused; views with gaps that are scaled
    where they lie may share it: all are read before anything is written, so that no element is scaled twice.  An infinite entry scales by zero and a NaN makes every
    gradient NaN.  Autograd records none of it.  With ``error_if_nonfinite`` a norm that is not finite in float32 raises RuntimeError and changes nothing
    (this waits for the GPU)."""
    p = _norm_type(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number that is not negative, got {max_norm}")
    grads = _list(grads)
    dst = grads if out is None else _list(out)
    if not grads and not dst:
        return grad_norm(grads, norm_type)
    if error_if_nonfinite:
        with torch.no_grad():
            norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}: they were not clipped")
    norm = _launch(grads, dst, p, max_norm) if grads else None
    if norm is not None:
        return norm
    if len(dst) != len(grads):
        raise ValueError(f"out has {len(dst)} tensors for {len(grads)} gradients")
    _check(grads, dst)
    # the kernels walk memory in order: a pair that lies differently, or with gaps, goes through contiguous copies
    src, to, back = list(grads), list(dst), []
    for i in _lib.torch_op("copied_pairs")(grads, dst):
        g, o = grads[i], dst[i]
        if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
            raise ValueError(_SHARED)
        src[i] = g.detach().resolve_neg().contiguous()
        to[i] = torch.empty(o.shape, dtype=o.dtype, device=o.device)
        back.append((o, to[i]))
    norm = _launch(src, to, p, max_norm)
    if norm is None:
        raise ValueError(_SHARED)
    with torch.no_grad():
        for o, t in back:
            o.copy_(t)
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """:func:`clip_grads` on the ``.grad`` of every parameter that has one, in place."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite=error_if_nonfinite)
