"""Rotary positions on the GPU: interleaved or half layout, all or part of the
head, plain or scaled for contexts longer than the trained one.

The reference rotates q and k with transformers' apply_rotary_pos_emb
(layer.py:66) from cos / sin tables made on the host side of every step.
Here a step hands over integer positions; frequencies are kept as 64-bit
fractions of a turn, so a position's phase is one exact integer product and
far positions lose no accuracy.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib
from ._tensors import (dtype_code, interleaved, launch, meets_itself, need_cuda, need_like, new_rows, overlap,
                       rows_of)

LAYOUTS = ("half", "interleaved")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_max_position: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> Tuple[Tensor, float]:
    """(freq, attention_factor) of rotary_dim / 2 pairs: freq int64, pair i's
    turns per position times 2^64; theta_i = base^(-2i / rotary_dim), scaled by

    * "linear": theta / factor (positions squeezed into the trained range);
    * "ntk": base grows to base * factor^(rd / (rd - 2)), so the slowest pair
      is squeezed by `factor` and the fastest keeps its pace;
    * "yarn": pairs that turn more than beta_fast times within
      original_max_position keep theta, those below beta_slow turns get
      theta / factor, with a linear ramp over the pairs between; rows are
      scaled by 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling={scaling}: none, linear, ntk or yarn")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError(f"base={base} must be above 1 and factor={factor} at least 1")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    theta = base ** (-2.0 * i / rotary_dim)
    attention_factor = 1.0
    if scaling == "linear":
        theta = theta / factor
    elif scaling == "yarn":
        if not original_max_position or original_max_position < 1:
            raise ValueError("yarn scaling needs original_max_position")

        def pair_of(turns):   # the (fractional) pair that turns `turns` times over the trained range
            return rotary_dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(pair_of(beta_fast)), 0)
        hi = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        theta = theta / factor * ramp + theta * (1 - ramp)
        attention_factor = 0.1 * math.log(factor) + 1.0
    turns = [round(t / (2 * math.pi) * 2.0 ** 64) for t in theta.tolist()]
    return torch.tensor(turns, dtype=torch.int64, device=device), attention_factor


def apply_rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, freq: Tensor, layout: str = "half",
                 attention_factor: float = 1.0, inverse: bool = False,
                 out: Optional[Tuple[Tensor, Optional[Tensor]]] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """Turn the first 2 * len(freq) channels of every row of q and k.

    q [n, Hq, D] and k [n, Hkv, D] with positions [n], or q [B, T, Hq, D] and
    k [B, T, Hkv, D] with positions [B, T] or [T]; any strides (transposed
    views are read in place), positions int32 or int64 of any sign, k may be
    None.  inverse turns back: it maps gradients of the results to gradients
    of the inputs, which is also what autograd gets (reverse mode, any order;
    forward mode and torch.func are not supported).  out = (q_out, k_out):
    tensors of the same shapes to write to (any strides with unit channel
    stride; they may lie in one buffer with each other and with the inputs, at
    other elements), new contiguous ones otherwise.
    """
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if out is not None:
            raise RuntimeError("apply_rotary: out= does not take part in autograd")
        return _Turn.apply(q, k, positions, freq, layout, attention_factor, inverse)
    return _turn(q, k, positions, freq, layout, attention_factor, inverse, out)


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freq, layout, attention_factor, inverse):
        # saved this way, a change of the positions before backward is an error
        ctx.save_for_backward(positions, freq)
        ctx.args = (layout, attention_factor, not inverse)
        return _turn(q, k, positions, freq, layout, attention_factor, inverse, None)

    @staticmethod
    def backward(ctx, dq, dk):
        # gradients of results that took no part come as zeros; differentiable again
        return (*apply_rotary(dq, dk, *ctx.saved_tensors, *ctx.args), None, None, None, None, None)


_NO_ROWS = (0, 0, 0, 0, 0, 0, 0, 0, 0)   # no tensor, no heads


def _rows(x: Tensor, y: Tensor):
    """carekv_rows_t of a row tensor and its result."""
    if x.dim() == 4:
        b, t, h, _ = x.stride()
        ob, ot, oh, _ = y.stride()
        return x.data_ptr(), y.data_ptr(), b, t, h, ob, ot, oh, x.shape[2]
    t, h, _ = x.stride()
    ot, oh, _ = y.stride()
    return x.data_ptr(), y.data_ptr(), 0, t, h, 0, ot, oh, x.shape[1]


def _check_out(q, k, positions, freq, out):
    yq, yk = out
    for x, y, what in ((q, yq, "q"), (k, yk, "k")):
        if (x is None) != (y is None):
            raise ValueError(f"apply_rotary out: one tensor for each of q and k ({what})")
        if x is None:
            continue
        need_like(y, q, f"apply_rotary out {what}")
        if y.shape != x.shape or (y.stride(-1) != 1 and x.shape[-1] > 1):
            raise ValueError(f"apply_rotary out {what}: expected shape {tuple(x.shape)} with unit channel stride")
        if y.numel() and meets_itself(y):
            raise ValueError(f"apply_rotary out {what}: its elements overlap one another")
        for t in (q, k, positions, freq) + ((yq,) if y is yk else ()):
            if t is not None and overlap(y, t) and not interleaved(y, t):
                raise ValueError("apply_rotary out: must not share storage elements with q, k, positions, freq or the "
                                 "other result")
    return yq, yk


def _turn(q, k, positions, freq, layout, attention_factor, inverse, out):
    need_cuda(q, "apply_rotary q")
    dt = dtype_code(q, "apply_rotary q")
    if layout not in LAYOUTS:
        raise ValueError(f"layout={layout}: half or interleaved")
    shape, nd = q.shape, q.dim()
    if nd != 3 and nd != 4:
        raise ValueError(f"apply_rotary q: expected [n, H, D] or [B, T, H, D], got {tuple(shape)}")
    D = shape[-1]
    batch, tokens = (shape[0], shape[1]) if nd == 4 else (1, shape[0])
    if k is not None:
        need_like(k, q, "apply_rotary k")
        ks = k.shape
        if len(ks) != nd or ks[0] != shape[0] or ks[-1] != D or (nd == 4 and ks[1] != tokens):
            raise ValueError(f"apply_rotary k: {tuple(ks)} does not match q {tuple(shape)}")
    index = q.get_device()
    if positions.get_device() != index or freq.get_device() != index:
        raise RuntimeError(f"apply_rotary: positions and freq belong on {q.device}")
    if positions.dtype is torch.int64:
        position_bytes = 8
    elif positions.dtype is torch.int32:
        position_bytes = 4
    else:
        raise ValueError(f"apply_rotary positions: int32 or int64, got {positions.dtype}")
    ps = positions.shape
    if len(ps) == 2 and nd == 4 and ps[0] == batch and ps[1] == tokens:
        sb, stok = positions.stride()
    elif len(ps) == 1 and ps[0] == tokens:
        sb, stok = 0, positions.stride(0)
    else:
        raise ValueError(f"apply_rotary positions: {tuple(ps)} does not match {tuple(shape[:-2])}")
    if freq.dtype is not torch.int64 or freq.dim() != 1 or not freq.is_contiguous():
        raise ValueError("apply_rotary freq: a contiguous int64 vector (rotary_frequencies)")
    rd = 2 * freq.shape[0]
    if not 0 < rd <= D:
        raise ValueError(f"apply_rotary: {rd} rotary channels do not fit a head of {D}")
    q = rows_of(q)
    if k is not None:
        k = rows_of(k)
    if out is not None:
        yq, yk = _check_out(q, k, positions, freq, out)
    else:
        yq = new_rows(q)
        yk = None if k is None else new_rows(k)
    args = _lib.ROTARY_PACK(*_rows(q, yq), *(_NO_ROWS if k is None else _rows(k, yk)), freq.data_ptr(),
                            positions.data_ptr(), sb, stok, position_bytes, batch, tokens, D, rd,
                            layout == "interleaved", bool(inverse), attention_factor, dt)
    launch(_lib.lib().carekv_rotary, q, "carekv_rotary", args)
    return yq, yk


class RotaryEmbedding(nn.Module):
    """Frequencies and layout of a model's rotary positions, kept on the device
    (a buffer that moves with the module and stays out of state dicts)."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_max_position: Optional[int] = None, device="cuda"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout={layout}: half or interleaved")
        super().__init__()
        self.layout = layout
        freq, self.attention_factor = rotary_frequencies(rotary_dim, base, scaling, factor, original_max_position,
                                                         device=device)
        self.register_buffer("freq", freq, persistent=False)

    def forward(self, q: Tensor, k: Optional[Tensor], positions: Tensor, inverse: bool = False, out=None):
        return apply_rotary(q, k, positions, self.freq, self.layout, self.attention_factor, inverse, out)
