"""4-bit weights with group scales for the projections of a decode step.

The codes and scales are the package quantizer's (``quantize`` with 4 bits,
``pack_int4_2d``); a PackedWeight holds them once more in the order in which
the product kernel's lanes read them, made when a model is loaded.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor, nn

from . import _lib
from ._tensors import DT, dtype_code, launch, need_cuda, need_like, overlap
from .quantizer import QuantConfig, pack_codes_2d, quantize

# Rows up to which matmul multiplies from the codes (PackedWeight.matmul).
# Measured, us on the device, codes against dequantize and the library's dense
# product: 13824 x 5120 (bf16) 64 rows 33 / 185, 128 rows 59 / 187, 256 88 / 191,
# 512 170 / 203, 1024 335 / 244; 1024 x 4096 (bf16) 64 rows 7 / 20, 192 19 / 20,
# 256 23 / 20; 4096 x 4096 (fp32) 64 rows 88 / 140, 128 173 / 165.  So the limit
# is on the safe side by a factor of about three in 16 bits and two in fp32.
MATVEC_ROWS = 64


class PackedWeight(nn.Module):
    """Weight [N, K] as 4-bit codes -8..7 times one scale per `group_size`
    channels of a row.  packed [N, K/2]: rows of ``pack_int4_2d``; scale
    [N, K/group_size] in the activations' dtype.  Codes and scales are byte
    buffers of the module, so state dicts hold them, copies and moves between
    devices keep them, and no cast changes them."""

    def __init__(self, packed: Tensor, scale: Tensor, group_size: int):
        super().__init__()
        need_cuda(packed, "PackedWeight packed")
        need_cuda(scale, "PackedWeight scale")
        if packed.dtype not in (torch.uint8, torch.int8) or packed.dim() != 2:
            raise ValueError(f"PackedWeight packed: expected a 2-d byte tensor, got {packed.dtype} "
                             f"{tuple(packed.shape)}")
        if scale.device != packed.device:
            raise RuntimeError(f"PackedWeight scale: expected a tensor on {packed.device}, got {scale.device}")
        n, k = packed.shape[0], 2 * packed.shape[1]
        if group_size < 1 or k % group_size or tuple(scale.shape) != (n, k // group_size):
            raise ValueError(f"PackedWeight: scale {tuple(scale.shape)} does not fit {n} rows of {k} channels in "
                             f"groups of {group_size}")
        packed, scale = packed.contiguous(), scale.contiguous()
        self.shape = (n, k)
        self.group_size = group_size
        self.dtype = scale.dtype
        c = _lib.W4(n=n, k=k, group_size=group_size, dtype=dtype_code(scale, "PackedWeight scale"))
        sizes = (ctypes.c_size_t * 2)()
        lib = _lib.lib()
        _lib.check(lib.carekv_w4_layout(ctypes.byref(c), sizes), "carekv_w4_layout")
        self.register_buffer("codes", torch.empty(sizes[0], dtype=torch.uint8, device=packed.device))
        self.register_buffer("scales", torch.empty(sizes[1], dtype=torch.uint8, device=packed.device))
        self._bind()
        launch(lib.carekv_w4_pack, packed, "carekv_w4_pack", self._ref, packed.data_ptr(), scale.data_ptr())

    def _bind(self):
        """The C structure of the buffers as they lie now; no device index off the GPU."""
        n, k = self.shape
        self.c = _lib.W4(self.codes.data_ptr(), self.scales.data_ptr(), n, k, self.group_size, DT[self.dtype])
        self._ref = ctypes.byref(self.c)
        self.device = self.codes.device
        self._index = self.codes.get_device() if self.codes.is_cuda and self.scales.device == self.device else None

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._bind()
        return self

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("c", "_ref")}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._bind()

    # What the bytes of a state dict stand for: another weight's may be as long.
    def get_extra_state(self):
        return dict(layout=1, shape=tuple(self.shape), group_size=self.group_size, dtype=str(self.dtype))

    def set_extra_state(self, state):
        pass   # compared before the buffers are read

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        held = state_dict.get(prefix + "_extra_state")
        if prefix + "codes" in state_dict and held != self.get_extra_state():
            error_msgs.append(f"PackedWeight {prefix}: expected {self.get_extra_state()}, got {held}")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)
        self._bind()

    @classmethod
    def from_dense(cls, weight: Tensor, group_size: int = 32) -> "PackedWeight":
        """Quantize a dense weight [N, K] with the package quantizer."""
        codes, scale = quantize(weight, QuantConfig(bits=4, group_size=group_size))
        return cls(pack_codes_2d(codes, 4), scale, group_size)

    def memory_bytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def matvec(self, x: Tensor, out: Optional[Tensor] = None) -> Tensor:
        """x [..., K] @ weight^T -> [..., N] in x's dtype (the scales' dtype),
        read from the codes: made for the few rows of a decode step.
        Differentiable in x (without out): its gradient is a dense product
        with the dequantized weight."""
        if x.requires_grad and torch.is_grad_enabled():
            if out is not None:
                raise RuntimeError("matvec: out= does not take part in autograd")
            return _Product.apply(x, self.codes, self.scales, self)
        n, k = self.shape
        if x.get_device() != self._index:
            need_cuda(self.codes, "PackedWeight")
            raise RuntimeError(f"matvec x: expected a tensor on {self.device}, got {x.device}")
        if x.dtype is not self.dtype:
            raise ValueError(f"matvec x: expected {self.dtype}, got {x.dtype}")
        shape = x.shape
        if not shape or shape[-1] != k:
            raise ValueError(f"matvec x: expected [..., {k}], got {tuple(shape)}")
        # rows the kernel can read in place: unit channel stride, every row
        # on a 16-byte boundary
        flat, plain = x, len(shape) == 2
        if plain:
            step, one = x.stride()
            plain = one == 1 and step >= k and step % 8 == 0
        if not plain:
            flat = x.reshape(-1, k).contiguous()
        if flat.data_ptr() % 16:
            flat = flat.clone(memory_format=torch.contiguous_format)
        rows = flat.shape[0]
        if out is None:
            out = x.new_empty((rows, n) if len(shape) == 2 else (*shape[:-1], n))
        else:
            need_like(out, x, "matvec out")
            if tuple(out.shape) != (*shape[:-1], n) or not out.is_contiguous():
                raise ValueError(f"matvec out: expected a contiguous tensor of shape {(*shape[:-1], n)}")
            if overlap(out, flat):
                raise ValueError("matvec out: must not overlap x")
        launch(_lib.lib().carekv_w4_matvec, x, "carekv_w4_matvec", self._ref, flat.data_ptr(),
               max(flat.stride(0), k), rows, out.data_ptr())
        return out

    def dequantize(self) -> Tensor:
        """The dense weight [N, K], codes * scale rounded to the scales' dtype."""
        need_cuda(self.codes, "PackedWeight")
        out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        launch(_lib.lib().carekv_w4_dequantize, out, "carekv_w4_dequantize", self._ref, out.data_ptr())
        return out

    def matmul(self, x: Tensor) -> Tensor:
        """x [..., K] @ weight^T for any number of rows: from the codes up to
        MATVEC_ROWS rows, with exact weights; above that (prompts) a dense
        product with the dequantized weight, whose entries are rounded to the
        dtype once (half an ulp each)."""
        if x.numel() <= MATVEC_ROWS * self.shape[1]:
            return self.matvec(x)
        return x @ self.dequantize().t()


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, weight):
        ctx.save_for_backward(codes, scales)   # a weight changed before backward is an error
        ctx.weight = weight
        return weight.matvec(x)   # with grad mode off

    @staticmethod
    def backward(ctx, dy):
        ctx.saved_tensors
        return dy @ ctx.weight.dequantize(), None, None, None
