"""Python entries to the gradient norm and clipping kernels (``csrc/kernels/clip.cu``).

Gradients are any number of contiguous f32, bf16 or f16 tensors of any size and alignment (views of a flat gradient vector among them). The norm is
that of all of them together, of ``scale`` times their values. Squares are summed in 64 bits above the first eight, in an order that the sizes
give. Each call launches on the current (or given) stream, can be captured into a graph and returns nothing."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _one(t: torch.Tensor | None, what: str) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != 1:
        raise ValueError(f"{what} must be one float32")
    return t.data_ptr()


def _clip(grads, outs, norm, coef, max_norm: float, scale: float, scratch, stream) -> None:
    if isinstance(grads, torch.Tensor) or isinstance(outs, torch.Tensor):
        raise TypeError("gradients come as a list of tensors")
    grads = list(grads)
    if not (max_norm > 0.0) or not math.isfinite(scale):
        raise ValueError("max_norm must be positive and scale finite")
    if outs is not None:
        outs = list(outs)
        if len(outs) != len(grads):
            raise ValueError("one output for each gradient")
        for g, o in zip(grads, outs):
            if o.shape != g.shape or o.dtype != g.dtype and o.data_ptr() == g.data_ptr() != 0:
                raise ValueError("an output has its gradient's shape, and over the gradient its type")
        at = [o.data_ptr() for o in outs if o.numel()]
        if len(set(at)) != len(at):
            raise ValueError("two outputs at one place")
    for t in grads if outs is None else grads + outs:
        if t.dtype not in _DTYPE:
            raise TypeError("gradients must be float32, bfloat16 or float16")
        if not t.is_contiguous():
            raise ValueError("gradients must be contiguous")
    home = norm if norm is not None else coef if coef is not None else grads[0] if grads else None
    if home is None:
        return
    _lib.one_device(home, *grads, *(outs or ()), norm, coef, scratch)
    lib = _lib.load()
    n = len(grads)
    arr = (_lib.OnoClipTensor * n)(*[
        (g.data_ptr(), None if outs is None else outs[k].data_ptr(), g.numel(), _DTYPE[g.dtype], 0 if outs is None else _DTYPE[outs[k].dtype])
        for k, g in enumerate(grads)])
    if scratch is None:
        scratch = _lib.scratch(home, lib.ono_clip_scratch(), stream)
    elif not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous")
    c = _lib.OnoClip(arr, n, scale, max_norm, _one(norm, "norm"), _one(coef, "coef"), outs is not None, scratch.data_ptr(),
                     scratch.numel() * scratch.element_size())
    _lib.launch(home, stream, "ono_clip", C.byref(c))


def clip_scratch() -> int:
    """Bytes of scratch that a call here wants."""
    return _lib.load().ono_clip_scratch()


def grad_norm(grads: list[torch.Tensor], norm: torch.Tensor, *, max_norm: float = math.inf, coef: torch.Tensor | None = None, scale: float = 1.0,
              scratch: torch.Tensor | None = None, stream=None) -> None:
    """``norm[0] = |scale| * sqrt(sum over all gradients of g^2)`` and, if wanted, ``coef[0]``, what clipping to ``max_norm`` multiplies the
    scaled gradients by: 1 up to ``max_norm``, ``max_norm / norm`` above (0 for an infinite norm, NaN for a NaN). ``elementwise.optim_step``
    takes it as ``grad_coef``: the step then clips as it goes, without a pass over the gradients."""
    _clip(grads, None, norm, coef, max_norm, scale, scratch, stream)


def clip_grads(grads: list[torch.Tensor], max_norm: float, *, scale: float = 1.0, norm: torch.Tensor | None = None,
               coef: torch.Tensor | None = None, out: list[torch.Tensor] | None = None, scratch: torch.Tensor | None = None, stream=None) -> None:
    """``out[k] = coef * scale * grads[k]`` (None: in place), coef as in ``grad_norm``, rounded once to the output's type: the gradients
    clipped together, into another type on the way if wanted (a 16-bit wire)."""
    grads = list(grads)
    _clip(grads, grads if out is None else out, norm, coef, max_norm, scale, scratch, stream)
