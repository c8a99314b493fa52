"""Python entries to the softmax over a vocabulary with one given token per row (``csrc/kernels/token_loss.cu``): log probabilities,
entropy, most likely alternatives, and the logits' gradients. ``elementwise.loss_backward`` is the form for one-hot (or soft) label rows.

Logits are 2-D rows with unit inner stride, f32 or bf16; targets int32 or int64, one a row. A gradient's ``out`` is the logits themselves or nowhere in them;
no other result lies in an input or in another result. Each call launches on the current (or given)
stream, can be captured into a graph and returns nothing.

A logit of -inf has probability zero. A row of nothing else has log probability and ``lse`` of -inf, entropy 0 and a gradient of zeros; a
row with a NaN or +inf has NaN for them. A row whose target is ``ignore_id`` (None: there is none) counts for nothing, whatever is in it:
zeros, and no alternatives. So does one whose target is outside the vocabulary, and then ``status`` (int32[1]) becomes non-zero."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._launch import DIM_MAX, id_or_none, launch, one_device, rows_of, status_ptr

_TARGETS = {torch.int32: 0, torch.int64: 1}

TOP_MAX = 32


def _column(t: torch.Tensor | None, rows: int, what: str) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != rows or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 vector of {rows} values")
    return t.data_ptr()


def _targets(t: torch.Tensor | None, rows: int) -> int:
    if t is None:
        return 0
    wide = _TARGETS.get(t.dtype)
    if wide is None:
        raise TypeError("targets must be int32 or int64")
    if t.dim() != 1 or t.shape[0] != rows or not t.is_contiguous():
        raise ValueError(f"targets must be a contiguous vector of {rows} values")
    return wide


def _logits(t: torch.Tensor) -> int:
    pitch = rows_of(t, "logits")
    if t.shape[1] > DIM_MAX:
        raise ValueError(f"a vocabulary has at most {DIM_MAX} tokens")
    return pitch


def _out(out: torch.Tensor, logits: torch.Tensor) -> int:
    pitch = rows_of(out, "out")
    if out.shape != logits.shape:
        raise ValueError("out must have the logits' shape")
    if out.data_ptr() == logits.data_ptr() and (out.dtype != logits.dtype or pitch != rows_of(logits, "logits")):
        raise ValueError("out over the logits needs the same type and rows")
    return pitch


def _tokens(logits, targets, ignore_id, status, stream, *, logp=None, lse=None, lse_low=None, entropy=None, top_logp=None, top_id=None, out=None, ld_out=0,
            weight=None, scale=1.0) -> None:
    ld = _logits(logits)
    rows, vocab = logits.shape
    wide = _targets(targets, rows)
    top = 0
    if top_logp is not None or top_id is not None:
        if top_logp is None or top_id is None or top_logp.dtype != torch.float32 or top_id.dtype != torch.int32:
            raise TypeError("top_logp (float32) and top_id (int32) go together")
        if top_logp.dim() != 2 or top_logp.shape != top_id.shape or top_logp.shape[0] != rows or not top_logp.is_contiguous() or not top_id.is_contiguous():
            raise ValueError(f"top_logp and top_id must be contiguous matrices of {rows} rows")
        top = top_logp.shape[1]
        if top > min(TOP_MAX, vocab):
            raise ValueError(f"at most {min(TOP_MAX, vocab)} alternatives")
    ignore_id = id_or_none(ignore_id)
    one_device(logits, targets, status, logp, lse, lse_low, entropy, top_logp, top_id, out, weight)
    a = _lib.OnoTokens(logits.data_ptr(), None if targets is None else targets.data_ptr(), rows, ld, ld_out, ignore_id,
                       vocab, logits.dtype == torch.bfloat16, wide, top, _column(logp, rows, "logp"), _column(lse, rows, "lse"),
                       _column(entropy, rows, "entropy"), top_logp.data_ptr() if top else None, top_id.data_ptr() if top else None,
                       None if out is None else out.data_ptr(), out is not None and out.dtype == torch.bfloat16, _column(weight, rows, "weight"),
                       scale, status_ptr(status), _column(lse_low, rows, "lse_low"))
    if rows == 0:
        return
    if vocab == 0:
        raise ValueError("logits of no tokens")
    launch(logits, stream, "ono_tokens", C.byref(a))


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None, *, logp: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                   lse_low: torch.Tensor | None = None, entropy: torch.Tensor | None = None, top_logp: torch.Tensor | None = None,
                   top_id: torch.Tensor | None = None, ignore_id: int | None = -1, status: torch.Tensor | None = None, stream=None) -> None:
    """With ``lse = ln sum_v exp(x_v)``: ``logp[r] = x[r, targets[r]] - lse[r]``, ``entropy[r] = -sum_v p_v ln p_v`` (natural logarithms, f32), and
    the ``top_id.shape[1]`` (at most ``TOP_MAX``) largest logits' tokens and log probabilities, the largest first and among equal ones
    the lowest token first. Where a row has fewer logits above -inf, id -1 and -inf follow. The logits are read once. Without ``targets`` every row
    counts and there is no ``logp``. ``lse_low``: what rounding to f32 took off ``lse``, for ``token_logprobs_grad``."""
    if targets is None and logp is not None:
        raise ValueError("logp needs targets")
    if lse_low is not None and lse is None:
        raise ValueError("lse_low needs lse")
    _tokens(logits, targets, ignore_id, status, stream, logp=logp, lse=lse, lse_low=lse_low, entropy=entropy, top_logp=top_logp, top_id=top_id)


def token_loss(logits: torch.Tensor, targets: torch.Tensor, *, out: torch.Tensor, logp: torch.Tensor | None = None,
               lse: torch.Tensor | None = None, weight: torch.Tensor | None = None, scale: float = 1.0, ignore_id: int | None = -1,
               status: torch.Tensor | None = None, stream=None) -> None:
    """The token cross entropy ``-scale * sum_r weight[r] * logp[r]`` by its gradient ``out = scale * weight[r] * (p - 1[v = target])`` (f32 or bf16;
    ``out`` may be ``logits``) and the rows' ``logp``, in one call: elementwise.loss_backward's counterpart for integer targets."""
    if targets is None:
        raise ValueError("a token loss needs targets")
    _tokens(logits, targets, ignore_id, status, stream, logp=logp, lse=lse, out=out, ld_out=_out(out, logits), weight=weight, scale=scale)


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor | None, *, lse: torch.Tensor, out: torch.Tensor,
                        d_logp: torch.Tensor | None = None, entropy: torch.Tensor | None = None, d_entropy: torch.Tensor | None = None,
                        lse_low: torch.Tensor | None = None, ignore_id: int | None = -1, status: torch.Tensor | None = None, stream=None) -> None:
    """The logits' gradient from those of ``token_logprobs``' results, ``lse`` and ``entropy`` being what it returned:
    ``out = d_logp (1[v = target] - p) - d_entropy p (ln p + entropy)``. ``out`` may be ``logits``.

    p is ``exp(logits - lse)``, so that half a step of ``lse`` is a relative error of a row's p: 4.8e-7 where ``lse`` is from 8 to 16, 3.8e-6 from 64 to 128 (beyond that
    the row's sum is taken again). A gradient in bf16 does not show it; for one in f32 give ``lse_low`` too, and p is as exact as ``token_loss`` has it."""
    ld = _logits(logits)
    rows, vocab = logits.shape
    wide = _targets(targets, rows)
    ld_out = _out(out, logits)
    if d_logp is None and d_entropy is None:
        raise ValueError("d_logp, d_entropy or both")
    if d_logp is not None and targets is None:
        raise ValueError("d_logp needs targets")
    if (entropy is None) != (d_entropy is None):
        raise ValueError("d_entropy needs the entropy, which has no other use")
    ignore_id = id_or_none(ignore_id)
    one_device(logits, targets, status, lse, lse_low, entropy, d_logp, d_entropy, out)
    a = _lib.OnoTokensGrad(logits.data_ptr(), None if targets is None else targets.data_ptr(), rows, ld, ld_out, ignore_id,
                           vocab, logits.dtype == torch.bfloat16, wide, _column(lse, rows, "lse"), _column(entropy, rows, "entropy"),
                           _column(d_logp, rows, "d_logp"), _column(d_entropy, rows, "d_entropy"), out.data_ptr(), out.dtype == torch.bfloat16,
                           status_ptr(status), _column(lse_low, rows, "lse_low"))
    if rows == 0 or vocab == 0:
        return
    launch(logits, stream, "ono_tokens_grad", C.byref(a))
