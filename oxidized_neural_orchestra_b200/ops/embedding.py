"""Python entries to the rows-by-token kernels (``csrc/kernels/embedding.cu``): a table's rows looked up by token, and its gradient.

Like the other ops each call launches on the current (or given) stream, can be captured into a graph and returns nothing. Tables and
rows are 2-D with unit inner stride, f32 or bf16; ids are int32 or int64, of any shape. What is written lies in none of the inputs."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._launch import DIM_MAX, id_or_none, launch, one_device, rows_of, scratch as scratch_for, status_ptr

_IDS = {torch.int32: 0, torch.int64: 1}


def _ids(ids: torch.Tensor, n: int) -> int:
    wide = _IDS.get(ids.dtype)
    if wide is None:
        raise TypeError("ids must be int32 or int64")
    if ids.numel() != n or not ids.is_contiguous():
        raise ValueError(f"ids must be contiguous, one for each of the {n} rows")
    return wide


def _sizes(vocab: int, width: int) -> None:
    if vocab > DIM_MAX or width > DIM_MAX:
        raise ValueError(f"a table has at most {DIM_MAX} rows and columns")


def embedding(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor, *, scale: float = 1.0, padding_id: int | None = -1,
              status: torch.Tensor | None = None, stream=None) -> None:
    """``out[i] = scale * table[ids[i]]`` (the product in f32, rounded once to the type of ``out``).

    An id equal to ``padding_id`` (None: there is none) stands for no token: its row is zeros. So is that of any other id
    outside the table, and then ``status`` (int32[1]) becomes non-zero."""
    ld_table, ld_out = rows_of(table, "table"), rows_of(out, "out")
    n, width = out.shape
    vocab = table.shape[0]
    wide = _ids(ids, n)
    if table.shape[1] != width:
        raise ValueError(f"table rows have {table.shape[1]} values, out rows {width}")
    _sizes(vocab, width)
    padding_id = id_or_none(padding_id)
    one_device(table, ids, out, status)
    if n == 0 or width == 0:
        return
    if vocab == 0:
        raise ValueError("a table without rows")
    e = _lib.OnoEmbedding(table.data_ptr(), ids.data_ptr(), out.data_ptr(), n, ld_table, ld_out, padding_id,
                          vocab, width, table.dtype == torch.bfloat16, out.dtype == torch.bfloat16, wide, scale, status_ptr(status))
    launch(table, stream, "ono_embedding", C.byref(e))


def embedding_grad_scratch(n: int, vocab: int, width: int) -> int:
    """Bytes of scratch that ``embedding_grad`` wants for ``n`` tokens (0 for few), and no more for any fewer of them."""
    _sizes(vocab, width)
    return _lib.load().ono_embedding_grad_scratch(n, vocab, width)


def embedding_grad(d: torch.Tensor, ids: torch.Tensor, grad: torch.Tensor, *, scale: float = 1.0, accumulate: bool = False,
                   padding_id: int | None = -1, scratch: torch.Tensor | None = None, status: torch.Tensor | None = None,
                   stream=None) -> None:
    """Gradient of the table behind ``embedding``: ``grad[v]`` (f32) becomes ``scale`` times the sum of the ``d[i]`` with ``ids[i] == v``,
    zeros for tokens that do not occur; with ``accumulate`` the sums are added to what is there and the other rows stay as they are. ``padding_id``
    and ``status`` as for ``embedding``.

    Sums are f32 and go over the places in one order that the sizes and the ids give: the same bits every time. ``scratch``: a
    contiguous tensor of at least ``embedding_grad_scratch`` bytes that no overlapping call uses (None: allocated for this call)."""
    ld_d, ld_grad = rows_of(d, "d"), rows_of(grad, "grad", (torch.float32,))
    n, width = d.shape
    vocab = grad.shape[0]
    wide = _ids(ids, n)
    if grad.shape[1] != width:
        raise ValueError(f"d rows have {width} values, grad rows {grad.shape[1]}")
    if scratch is not None and not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous")
    _sizes(vocab, width)
    padding_id = id_or_none(padding_id)
    one_device(d, ids, grad, status, scratch)
    if vocab == 0 or width == 0:
        return
    if scratch is None:
        need = _lib.load().ono_embedding_grad_scratch(n, vocab, width)
        if need:
            scratch = scratch_for(grad, need, stream)
    e = _lib.OnoEmbeddingGrad(d.data_ptr(), ids.data_ptr(), grad.data_ptr(), n, ld_d, ld_grad, padding_id,
                              vocab, width, d.dtype == torch.bfloat16, wide, accumulate, scale, status_ptr(status),
                              None if scratch is None else scratch.data_ptr(), 0 if scratch is None else scratch.numel() * scratch.element_size())
    launch(grad, stream, "ono_embedding_grad", C.byref(e))
