"""The norm over all gradients of a model, and clipping (``disco_grad_norm`` / ``disco_grad_clip``).

Any number of tensors, float32 / float16 / bfloat16 in any mixture, in two or three launches; the norm stays on the device,
nothing synchronises.  No counterpart in the reference, whose training loops do not clip
(/root/reference/LargeScaleCondensing.py:187-200).  There is no CPU fallback.
"""
from __future__ import annotations

import math
from array import array
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib

_NORMS = {1.0: 1, 2.0: 2, math.inf: 0}
_SHARED = "clip_grads: two tensors share memory; each gradient may be scaled only once"


def _tensors(grads) -> List[torch.Tensor]:
    """The list of gradients.  The checks go list by list rather than tensor by tensor: a model has hundreds of them."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        return grads
    if not all([isinstance(g, torch.Tensor) for g in grads]):
        raise TypeError("gradients must be dense tensors")
    kinds = {(g.layout, g.dtype, g.device) for g in grads}
    if len(kinds) == 1 and grads[0].layout is torch.strided and grads[0].dtype in _lib.DTYPES:
        return grads
    if any([layout is not torch.strided for layout, _, _ in kinds]):
        raise TypeError("gradients must be dense tensors")
    if not {dtype for _, dtype, _ in kinds} <= _lib.DTYPES.keys():
        raise TypeError(f"gradients must be float32, float16 or bfloat16, got {sorted({str(dtype) for _, dtype, _ in kinds})}")
    if len({device for _, _, device in kinds}) > 1:
        raise ValueError(f"gradients on {sorted({str(device) for _, _, device in kinds})}: one device at a time")
    return grads


def _on_gpu(grads) -> None:
    if grads and not grads[0].is_cuda:
        raise RuntimeError(f"gradients on {grads[0].device}: disco_amd runs on the GPU only, there is no CPU fallback")


def _norm_type(norm_type) -> int:
    p = _NORMS.get(float(norm_type))
    if p is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type!r}")
    return p


def _codes(tensors) -> array:
    codes = _lib.DTYPES
    return array("i", [codes[t.dtype] for t in tensors])


def _launch(grads: Sequence[torch.Tensor], p: int, max_norm: Optional[float], out) -> torch.Tensor:
    first = grads[0]
    index = first.get_device()
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _launch(grads, p, max_norm, out)
    lib = _lib.load()
    n = len(grads)
    src = array("Q", [g.data_ptr() for g in grads])
    numel = array("q", [g.numel() for g in grads])
    types = _codes(grads)
    nb = lib.disco_grad_norm_workspace_bytes(n)
    ws = torch.empty(nb, dtype=torch.uint8, device=first.device)
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    stream = _lib.stream_of(index)
    if max_norm is None:
        status = lib.disco_grad_norm(src.buffer_info()[0], numel.buffer_info()[0], types.buffer_info()[0], n, p, norm.data_ptr(),
                                     ws.data_ptr(), nb, stream)
        _lib.check(status, "disco_grad_norm")
    else:
        same = out is grads
        dst = src if same else array("Q", [o.data_ptr() for o in out])
        to = types if same else _codes(out)
        status = lib.disco_grad_clip(src.buffer_info()[0], dst.buffer_info()[0], numel.buffer_info()[0], types.buffer_info()[0],
                                     to.buffer_info()[0], n, p, max_norm, norm.data_ptr(), ws.data_ptr(), nb, stream)
        if status == -1:
            raise ValueError(_SHARED)
        _lib.check(status, "disco_grad_clip")
        # written behind autograd's back: whoever saved one of them must notice
        try:
            torch.autograd.graph.increment_version(out)
        except RuntimeError:      # tensors made in inference mode keep no version
            torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
    return norm


def _dense(g: torch.Tensor) -> bool:
    """Elements fill one block of memory, in any order of the dimensions: the kernels may walk it as it lies."""
    if g.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(((n, s) for n, s in zip(g.shape, g.stride()) if n > 1), key=lambda d: d[1]):
        if stride != expected:
            return False
        expected *= size
    return True


def grad_norm(grads: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """``(sum |g|^p)^(1/p)`` over every element of every tensor, p = ``norm_type`` in {1, 2, inf}; a float32 scalar on the
    device.  Sums run in float64 in a fixed order: nothing overflows in between, and the result does not vary."""
    p = _norm_type(norm_type)
    grads = _tensors(grads)
    _on_gpu(grads)
    if not grads:
        return torch.zeros((), dtype=torch.float32, device="cuda" if torch.cuda.is_available() else "cpu")
    return _launch([g if _dense(g) else g.detach().contiguous() for g in grads], p, None, None)


def clip_grads(grads: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales every gradient by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm before (float32, on the device).

    In place by default; ``out`` names one destination per gradient, of its shape and either its type or float32 (the
    buffers a mixed-precision optimiser reads).  Tensors that share memory are refused.  An infinite norm scales by zero
    and a NaN norm makes every gradient NaN; with ``error_if_nonfinite`` such a norm raises RuntimeError and changes
    nothing (this waits for the GPU)."""
    p = _norm_type(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number that is not negative, got {max_norm}")
    grads = _tensors(grads)
    if out is None:
        dst = grads
    else:
        dst = _tensors(out)
        if len(dst) != len(grads):
            raise ValueError(f"out has {len(dst)} tensors for {len(grads)} gradients")
        f32 = torch.float32
        if dst and dst[0].device != grads[0].device or any(
                [o.shape != g.shape or (o.dtype is not f32 and o.dtype is not g.dtype) for g, o in zip(grads, dst)]):
            for g, o in zip(grads, dst):
                if o.shape == g.shape and o.device == g.device and o.dtype in (g.dtype, f32):
                    continue
                raise ValueError(f"out must have the gradients' shapes and device and their type or float32, got {tuple(o.shape)} "
                                 f"{o.dtype} on {o.device} for {tuple(g.shape)} {g.dtype} on {g.device}")
    _on_gpu(grads)
    if not grads:
        return grad_norm(grads, norm_type)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}: they were not clipped")
    if all([o.is_contiguous() for o in dst]) and (dst is grads or all([g.is_contiguous() for g in grads])):
        return _launch(grads, p, max_norm, dst)
    # the kernels walk memory in order: a pair that lies differently, or with gaps, goes through contiguous copies
    src, to, back = [], [], []
    for g, o in zip(grads, dst):
        if _dense(o) and (o is g or (_dense(g) and o.stride() == g.stride())):
            src.append(g)
            to.append(o)
            continue
        if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
            raise ValueError(_SHARED)
        src.append(g.detach().contiguous())
        to.append(torch.empty(o.shape, dtype=o.dtype, device=o.device))
        back.append((o, to[-1]))
    norm = _launch(src, p, max_norm, to)
    with torch.no_grad():
        for o, t in back:
            o.copy_(t)
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """:func:`clip_grads` on the ``.grad`` of every parameter that has one, in place."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite=error_if_nonfinite)
