"""Checks and launch plumbing shared by the tensor-level operators."""

import contextlib

import torch

from . import _lib

DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_SAME = contextlib.nullcontext()


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DT.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: unsupported dtype {t.dtype}")
    return code


def need_cuda(t: torch.Tensor, what: str):
    if not t.is_cuda:
        raise RuntimeError(f"{what}: the B200 build runs on CUDA tensors only (got {t.device})")


def need_like(t: torch.Tensor, like: torch.Tensor, what: str):
    """Same device and dtype as `like`."""
    if t.get_device() != like.get_device():
        raise RuntimeError(f"{what}: expected a tensor on {like.device}, got {t.device}")
    if t.dtype != like.dtype:
        raise ValueError(f"{what}: expected {like.dtype}, got {t.dtype}")


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride along its last dimension (a copy where it has another)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def new_rows(t: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(tuple(t.shape))


def on_device(t: torch.Tensor):
    """Context in which t's device is current (nothing to do when it is)."""
    return _SAME if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def stream(t: torch.Tensor) -> int:
    """Handle of the current stream of t's device.  The raw getter takes 0.07 us
    where building a torch Stream object takes 2.2 us, which counts in a call
    whose kernel runs for 3 us."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())
