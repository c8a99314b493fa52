"""What the operators on tokens, on gradients and of the optimizer share on the host: their checks, their scratch memory and the launch itself. A call of theirs may
take the GPU a few microseconds, so nothing here costs more than it has to."""
from __future__ import annotations

import torch

from . import _lib

DIM_MAX = 2**31 - 2**16      # rows' lengths and tables' rows: the kernels count them in 32 bits, some a block's stride beyond the last
NO_ID = -(2**63)


def id_or_none(value: int | None) -> int:
    """An id that stands for no token, or one that no ids have."""
    if value is None:
        return NO_ID
    if not NO_ID < value < -NO_ID:
        raise ValueError(f"no id is {value}")
    return value


def one_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """All on one GPU (None among them does not count)."""
    if not first.is_cuda:
        raise RuntimeError("this op runs on CUDA only (no CPU fallback on this path)")
    at = first.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise ValueError(f"tensors on different devices: cuda:{at} and {t.device}")


def rows_of(t: torch.Tensor, what: str, dtypes=(torch.float32, torch.bfloat16)) -> int:
    """Elements from one row of a matrix to the next, which has to have unit inner stride and rows one behind the other."""
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}")
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D")
    rows, width = t.shape
    pitch, step = t.stride()
    if step != 1 and width > 1 or pitch < width and rows > 1:
        raise ValueError(f"{what} must be rows with unit inner stride")
    return pitch if rows > 1 else width


def status_ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() < 1:
        raise TypeError("status must be int32")
    return t.data_ptr()


def scratch(t: torch.Tensor, nbytes: int, stream) -> torch.Tensor:
    """Memory for one call that launches on ``stream`` (None: the current one) of the GPU of ``t``: the allocator gives it to nobody else
    before what that stream holds now has run."""
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=t.device)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=t.device)


def launch(t: torch.Tensor, stream, name: str, *args) -> None:
    """``name(*args, stream)`` with the GPU of ``t`` as the current device, on ``stream`` (None: the one that is current there)."""
    fn, at = getattr(_lib.load(), name), t.get_device()
    if at == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(at) if stream is None else stream.cuda_stream)
    else:
        with torch.cuda.device(at):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(at) if stream is None else stream.cuda_stream)
    if rc:
        _lib.check(rc, name)
