"""Python entries to the gradient norm and clipping kernels (``csrc/kernels/clip.cu``).

Gradients are any number of contiguous f32, bf16 or f16 tensors of any size and alignment (views of a flat gradient vector among them); what is
written overlaps neither another output nor another gradient. The norm is that of all of them together, of ``scale`` times their values. Squares are
summed in 64 bits above the first eight, in an order that sizes and alignment give. Each call launches on the current (or given) stream, can be
captured into a graph and returns nothing."""
from __future__ import annotations

import ctypes as C
import math
from array import array

import torch

from . import _lib
from ._launch import launch, one_device, scratch as scratch_for

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# Hundreds of tensors are common. What is asked of all of them is asked by map, which takes two thirds of the time of a loop.
_CONTIGUOUS, _AT, _SIZE, _DEVICE = torch.Tensor.is_contiguous, torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device


def _types(ts: list[torch.Tensor]) -> bytes:
    if not all(map(_CONTIGUOUS, ts)):
        raise ValueError("gradients must be contiguous")
    kinds = {t.dtype for t in ts}
    if not kinds <= _DTYPE.keys():
        raise TypeError("gradients must be float32, bfloat16 or float16")
    return bytes([_DTYPE[t.dtype] for t in ts]) if len(kinds) > 1 else bytes([_DTYPE[k] for k in kinds]) * len(ts)


def _mixed(types: bytes, out_types: bytes) -> bytes:
    if len(types) and types == types[:1] * len(types) and out_types == out_types[:1] * len(types):
        return bytes([types[0] | out_types[0] << 2]) * len(types)
    return bytes([i | j << 2 for i, j in zip(types, out_types)])


def _one(t: torch.Tensor | None, what: str) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != 1:
        raise ValueError(f"{what} must be one float32")
    return t.data_ptr()


def _clip(grads, outs, write: bool, norm, coef, max_norm: float, scale: float, scratch, stream) -> None:
    if isinstance(grads, torch.Tensor) or isinstance(outs, torch.Tensor):
        raise TypeError("gradients come as a list of tensors")
    grads = list(grads)
    if not (max_norm > 0.0) or not math.isfinite(scale):
        raise ValueError("max_norm must be positive and scale finite")
    types, at, sizes, n = _types(grads), list(map(_AT, grads)), list(map(_SIZE, grads)), len(grads)
    to, out_types = [], types
    if write:
        if outs is None:
            to = at
        else:
            outs = list(outs)
            if len(outs) != n:
                raise ValueError("one output for each gradient")
            out_types, to = _types(outs), list(map(_AT, outs))
            if list(map(_SIZE, outs)) != sizes:
                raise ValueError("an output has as many values as its gradient")
            if types != out_types and any([p == q != 0 and i != j for p, q, i, j in zip(at, to, types, out_types)]):
                raise ValueError("an output over its gradient has the gradient's type")
        there = to if all(to) else [p for p in to if p]
        if len(set(there)) != len(there):
            raise ValueError("two outputs at one place")
    home = norm if norm is not None else coef if coef is not None else grads[0] if grads else None
    if home is None:
        return
    one_device(home, norm, coef, scratch)
    if not {home.get_device()}.issuperset(map(_DEVICE, grads)) or outs and not {home.get_device()}.issuperset(map(_DEVICE, outs)):
        raise ValueError("tensors on different devices")
    if scratch is None:
        scratch = scratch_for(home, clip_scratch(), stream)
    elif not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous")
    words = [array("q", v) for v in (at, to, sizes)]
    c = _lib.OnoClip(n, words[0].buffer_info()[0], words[1].buffer_info()[0] if write else None, words[2].buffer_info()[0], _mixed(types, out_types),
                     scale, max_norm, _one(norm, "norm"), _one(coef, "coef"), scratch.data_ptr(), scratch.numel() * scratch.element_size())
    launch(home, stream, "ono_clip", C.byref(c))


def clip_scratch() -> int:
    """Bytes of scratch that a call here wants."""
    return _lib.load().ono_clip_scratch()


def grad_norm(grads: list[torch.Tensor], norm: torch.Tensor, *, max_norm: float = math.inf, coef: torch.Tensor | None = None, scale: float = 1.0,
              scratch: torch.Tensor | None = None, stream=None) -> None:
    """``norm[0] = |scale| * sqrt(sum over all gradients of g^2)`` and, if wanted, ``coef[0]``, what clipping to ``max_norm`` multiplies the
    scaled gradients by: 1 up to ``max_norm``, ``max_norm / norm`` above (0 for an infinite norm, NaN for a NaN). ``elementwise.optim_step``
    takes it as ``grad_coef``: the step then clips as it goes, without a pass over the gradients."""
    _clip(grads, None, False, norm, coef, max_norm, scale, scratch, stream)


def clip_grads(grads: list[torch.Tensor], max_norm: float, *, scale: float = 1.0, norm: torch.Tensor | None = None,
               coef: torch.Tensor | None = None, out: list[torch.Tensor] | None = None, scratch: torch.Tensor | None = None, stream=None) -> None:
    """``out[k] = coef * scale * grads[k]`` (None: in place; else as many values, in their order), coef as in ``grad_norm``, rounded once to the output's type: the gradients
    clipped together, into another type on the way if wanted (a 16-bit wire)."""
    _clip(grads, out, True, norm, coef, max_norm, scale, scratch, stream)
