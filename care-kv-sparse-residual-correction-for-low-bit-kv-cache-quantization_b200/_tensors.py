"""Checks and launch plumbing shared by the tensor-level operators."""

import torch

from . import _lib

DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


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


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors (non-negative strides) meet."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(
        (n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b))
    return a0 < b1 and b0 < a1


def interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors whose address ranges meet have no element in common for
    this reason: they repeat with the same outer sizes and strides, and one
    repetition of both lies within a stride with its ranges apart (slices of
    one fused buffer)."""
    (ap, ad), (bp, bd) = ((t.data_ptr(), sorted(((s * t.element_size(), n) for n, s in zip(t.shape, t.stride()) if n > 1),
                                                reverse=True)) for t in (a, b))
    ea, eb = ([t.element_size() + sum((n - 1) * s for s, n in d[i:]) for i in range(len(d) + 1)]
              for t, d in ((a, ad), (b, bd)))
    for i in range(min(len(ad), len(bd)) + 1):
        if ap + ea[i] <= bp or bp + eb[i] <= ap:
            return True
        if i == min(len(ad), len(bd)) or ad[i] != bd[i]:
            return False
        if max(ap + ea[i + 1], bp + eb[i + 1]) - min(ap, bp) > ad[i][0]:
            return False
    return False


def meets_itself(t: torch.Tensor) -> bool:
    """Whether an axis steps into the elements of the axes within it (as an
    expanded one does)."""
    end = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < end:
            return True
        end += (n - 1) * s
    return False


def launch(fn, t: torch.Tensor, where: str, *args):
    """fn(*args, stream) with t's device current and on its current stream;
    raises on a status other than 0.  The raw getters take 0.1 us where
    torch.cuda.current_stream takes 2.2 us, which counts in a call whose
    kernel runs for 3 us."""
    index = t.get_device()
    if index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, where)


def check_operator_errors(device=None):
    """Raises if a wait inside a 4-bit product or a shared-prefix attention on
    the device (default: the current one) ran out since the last check; such a
    call's rows are NaN.  Synchronizes the device's current stream."""
    with torch.cuda.device(device):
        _lib.check(_lib.lib().carekv_check_operator_errors(None, torch.cuda.current_stream().cuda_stream),
                   "operator check")
