"""Attention of a whole batch over one shared prompt prefix.

Sequences that start with the same prompt hold its K / V once, at full
precision, instead of once per sequence in the packed arena: its bytes are
shared by the batch, so quantizing them would save little, and every tile is
read once per step for all sequences.  The sequences' own tokens stay in the
arena; ``DecodeEngine.attend(..., prefix=...)`` merges both.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._tensors import dtype_code, launch, need_cuda, need_like, new_rows, overlap, rows_of


def prefix_attention(q: Tensor, k: Tensor, v: Tensor, scale: Optional[float] = None,
                     lengths: Optional[Tensor] = None, tail: Optional[Tuple[Tensor, Tensor]] = None,
                     out: Optional[Tensor] = None, return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """softmax(scale q K^T) V of every row over the prefix, merged with the
    rows' own attention state.

    q [n, Hq, D]; k, v [Hkv, N, D] (Hq a multiple of Hkv; any strides with
    unit channel stride; N may be 0); scale > 0 defaults to 1 / sqrt(D).  lengths
    [n] int32: row r sees the prefix tokens below lengths[r] (clamped to
    0..N).  tail = (o [n, Hq, D], lse [n, Hq] fp32): attention output and
    natural log-sum-exp of the row's own tokens, -inf where it has none.
    out: a contiguous tensor to write to that overlaps no input, but may be
    tail's o itself.
    Returns [n, Hq, D] in q's dtype, with return_lse also the merged
    log-sum-exp [n, Hq] fp32; a row that sees nothing gives 0 and -inf.
    Values of a token that any row sees must be finite for every row.
    fp16 / bf16 with D 64 or 128 run on the tensor cores, with the softmax
    weights rounded to that type for the product with V; fp32, other D, and
    q, k, v, out or tail rows that do not start on 16-byte boundaries take an
    fp32 form that is about 100 times slower on long prefixes.
    There is no backward pass: inputs that require a gradient are refused.
    """
    if (q.requires_grad or k.requires_grad or v.requires_grad or (
            tail is not None and (tail[0].requires_grad or tail[1].requires_grad))) and torch.is_grad_enabled():
        raise RuntimeError("prefix_attention has no backward pass: detach its inputs or call it under no_grad")
    need_cuda(q, "prefix_attention q")
    dt = dtype_code(q, "prefix_attention q")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"prefix_attention: expected q [n, Hq, D] and k, v [Hkv, N, D], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    n, hq, d = q.shape
    hkv, tokens, dk = k.shape
    need_like(k, q, "prefix_attention k")
    need_like(v, q, "prefix_attention v")
    if dk != d or v.shape != k.shape:
        raise ValueError(f"prefix_attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"prefix_attention: {hq} query heads over {hkv} kv heads")
    q, k, v = rows_of(q), rows_of(k), rows_of(v)
    if lengths is not None:
        if lengths.get_device() != q.get_device() or lengths.dtype is not torch.int32 or lengths.dim() != 1 \
                or lengths.shape[0] != n:
            raise ValueError(f"prefix_attention lengths: expected int32 [{n}] on {q.device}")
        lengths = lengths.contiguous()
    tail_o = tail_lse = None
    if tail is not None:
        tail_o, tail_lse = tail
        need_like(tail_o, q, "prefix_attention tail output")
        if tail_o.shape != q.shape or tail_lse.shape != q.shape[:2] or tail_lse.dtype is not torch.float32 \
                or tail_lse.get_device() != q.get_device():
            raise ValueError("prefix_attention tail: expected (output like q, fp32 log-sum-exp [n, Hq])")
        tail_o, tail_lse = tail_o.contiguous(), tail_lse.contiguous()
    if out is None:
        out = new_rows(q)
    else:
        need_like(out, q, "prefix_attention out")
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"prefix_attention out: expected a contiguous tensor of shape {tuple(q.shape)}")
        # a row's own state is read by the threads that write the row: in place is fine
        others = [t for t in (q, k, v, lengths, tail_lse) if t is not None]
        if tail_o is not None and tail_o.data_ptr() != out.data_ptr():
            others.append(tail_o)
        if any(overlap(out, t) for t in others):
            raise ValueError("prefix_attention out: must not overlap its inputs (but may be the own state's output)")
    lse = q.new_empty((n, hq), dtype=torch.float32) if return_lse else None
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    prefix = _lib.PREFIX_PACK(k.data_ptr(), v.data_ptr(), k0, k1, v0, v1, hkv, tokens, d, dt)
    index = q.get_device()
    need = _workspace_bytes(n, hq, hkv, tokens, d, dt, index)
    ws = torch.empty(need, dtype=torch.uint8, device=index) if need else None
    row, head, _ = q.stride()
    launch(_lib.lib().carekv_prefix_attention, q, "carekv_prefix_attention", prefix, q.data_ptr(), row, head, n, hq,
           1.0 / math.sqrt(d) if scale is None else scale, None if lengths is None else lengths.data_ptr(),
           None if tail_o is None else tail_o.data_ptr(), None if tail_lse is None else tail_lse.data_ptr(),
           out.data_ptr(), None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), need)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(n, hq, hkv, tokens, d, dt, device) -> int:
    """Workspace of a shape on a device (its number of SMs enters)."""
    need = ctypes.c_size_t(0)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().carekv_prefix_workspace_bytes(_lib.PREFIX_PACK(0, 0, 0, 0, 0, 0, hkv, tokens, d, dt), n,
                                                            hq, ctypes.byref(need)), "carekv_prefix_workspace_bytes")
    return need.value


class SharedPrefix:
    """K / V of one prompt prefix for every layer, post-RoPE at positions
    0 .. tokens - 1, shared by all sequences of a cache."""

    def __init__(self, num_layers: int):
        self._kv = [None] * num_layers

    def set(self, layer: int, k: Tensor, v: Tensor):
        """k, v [Hkv, N, D] of one layer (copied).  A layer may be set anew; all
        layers hold the same number of tokens."""
        if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"SharedPrefix: k {tuple(k.shape)} and v {tuple(v.shape)} must match")
        self._kv[layer]   # an index that there is
        n = next((kv[0].shape[1] for i, kv in enumerate(self._kv)
                  if kv is not None and i != layer % len(self._kv)), None)
        if n is not None and k.shape[1] != n:
            raise ValueError(f"SharedPrefix: layer {layer} holds {k.shape[1]} tokens, the others {n}")
        self._kv[layer] = tuple(t.detach().clone(memory_format=torch.contiguous_format) for t in (k, v))

    @property
    def tokens(self) -> Optional[int]:
        """Tokens of the prefix (None before any layer is set)."""
        return next((kv[0].shape[1] for kv in self._kv if kv is not None), None)

    def layer(self, layer: int) -> Tuple[Tensor, Tensor]:
        kv = self._kv[layer]
        if kv is None:
            raise ValueError(f"SharedPrefix: layer {layer} has not been set")
        return kv

    def check(self, layer: int, kv_heads: int, head_dim: int, dtype: torch.dtype):
        """Raises unless the layer is set, to that many kv heads of that size and dtype."""
        k, _ = self.layer(layer)
        if k.dtype != dtype or k.shape[0] != kv_heads or k.shape[2] != head_dim:
            raise ValueError(f"SharedPrefix: expected {dtype} [{kv_heads}, tokens, {head_dim}] as the cache's kv heads, "
                             f"got {k.dtype} {tuple(k.shape)}")

    def memory_bytes(self) -> int:
        return sum(2 * kv[0].numel() * kv[0].element_size() for kv in self._kv if kv is not None)

    def attend(self, layer: int, q: Tensor, **kw):
        """prefix_attention of q [n, Hq, D] over this layer's prefix."""
        k, v = self.layer(layer)
        return prefix_attention(q, k, v, **kw)
