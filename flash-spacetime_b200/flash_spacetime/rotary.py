"""Rotary positions for q and k, before an attention op of this package.

``flash_rotary`` (padded) and ``flash_rotary_varlen`` (packed) rotate the
channel pairs of q and k by ``position * freqs`` in one launch of
``fst_rotary``; ``reference.rotary_frequencies`` makes the frequencies. The
gradient is the rotation by the opposite angle, so nothing of q and k is kept
for the backward.
"""

import struct
from typing import Any, Optional, Tuple

import torch
from torch import Tensor

from .grouped import (_CONTIGUOUS, _NO_ROWS, _ROWS, _call, _check_tensor, _finite_fp32, _int32,
                      _integers, _rows, _shape, once, seen_by_autograd)
from .ops import _DTYPES

_ROTARY = struct.Struct("@11ifq3Q" + 4 * _ROWS)


def _adjacent(t: Tensor) -> Tensor:
    """``t``, copied if a head's channels are not adjacent."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rotate(q: Tensor, k: Optional[Tensor], freqs: Tensor, cu: Optional[Tensor],
            positions: Optional[Tensor], layout: str, interleaved: bool, magnitude: float,
            inverse: bool) -> Tuple[Tensor, Optional[Tensor]]:
    """One ``fst_rotary`` call."""
    q = _adjacent(q)
    q_out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    events, rows, heads, dim = _shape(q, layout, "q")
    k_out, kv_heads, k_rows, k_out_rows = None, 0, _NO_ROWS, _NO_ROWS
    if k is not None:
        k = _adjacent(k)
        k_out = torch.empty_like(k, memory_format=_CONTIGUOUS)
        kv_heads, k_rows, k_out_rows = _shape(k, layout, "k")[2], _rows(k, layout), _rows(k_out, layout)
    packed = layout == "packed"
    batch = (0 if cu is None else cu.shape[0] - 1) if packed else events
    args = _ROTARY.pack(
        _DTYPES[q.dtype], packed, batch, heads, kv_heads, 0 if packed else rows, dim,
        freqs.shape[0], interleaved, inverse,
        positions is not None and positions.dtype == torch.int64, magnitude,
        rows if packed else events * rows, freqs.data_ptr(), 0 if cu is None else cu.data_ptr(),
        0 if positions is None else positions.data_ptr(), *_rows(q, layout), *k_rows,
        *_rows(q_out, layout), *k_out_rows)
    _call("fst_rotary", args, q.device)
    return q_out, k_out


class _FlashRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Optional[Tensor], freqs: Tensor, cu: Optional[Tensor],
                positions: Optional[Tensor], layout: str, interleaved: bool,
                magnitude: float) -> Tuple[Tensor, Optional[Tensor]]:  # type: ignore[override]
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(freqs, cu, positions)
        ctx.how = (layout, interleaved, magnitude)
        return _rotate(q, k, freqs, cu, positions, layout, interleaved, magnitude, False)

    @staticmethod
    def backward(ctx: Any, gq: Optional[Tensor], gk: Optional[Tensor]):  # type: ignore[override]
        return once(_backward)(ctx, gq, gk)


def _backward(ctx: Any, gq: Optional[Tensor], gk: Optional[Tensor]) -> Tuple[Any, ...]:
    freqs, cu, positions = ctx.saved_tensors
    layout, interleaved, magnitude = ctx.how
    gq = gq if ctx.needs_input_grad[0] else None
    gk = gk if ctx.needs_input_grad[1] else None
    dq = dk = None
    if gq is not None:
        dq, dk = _rotate(gq, gk, freqs, cu, positions, layout, interleaved, magnitude, True)
    elif gk is not None:
        dk, _ = _rotate(gk, None, freqs, cu, positions, layout, interleaved, magnitude, True)
    return dq, dk, None, None, None, None, None, None


def _apply(q: Tensor, k: Optional[Tensor], freqs: Tensor, cu: Optional[Tensor],
           positions: Optional[Tensor], layout: str, interleaved: bool,
           magnitude: float) -> Tuple[Tensor, Optional[Tensor]]:
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    events, rows, heads, dim = _shape(q, layout, "q")
    _check_tensor(q, q, "q")
    if k is not None:
        _check_tensor(k, q, "k")
        if _shape(k, layout, "k")[:2] != (events, rows) or k.shape[-1] != dim:
            raise ValueError(f"k {tuple(k.shape)} must have q's events, rows and Dh, q is "
                             f"{tuple(q.shape)}")
        if _shape(k, layout, "k")[2] < 1:
            raise ValueError("k has no heads (pass k=None)")
    if heads < 1 or not 1 <= dim <= 1024:
        raise ValueError(f"q must have heads of 1 to 1024 channels, got {tuple(q.shape)}")
    if not isinstance(freqs, Tensor):
        raise ValueError(f"freqs must be a tensor, got {type(freqs).__name__}")
    if layout != "packed" and rows >= 2**31:
        raise ValueError(f"{rows} rows an event: at most {2**31 - 1}")
    if freqs.dim() != 1 or not freqs.dtype.is_floating_point or 2 * freqs.numel() > dim:
        raise ValueError(f"freqs must be [R/2] floats with R <= Dh (={dim}), got "
                         f"{tuple(freqs.shape)} {freqs.dtype}")
    if freqs.requires_grad:
        raise ValueError("freqs must not require grad")
    freqs = freqs.to(device=q.device, dtype=torch.float64).contiguous()
    if positions is not None:
        _integers(positions, "positions")
        want = (rows,) if layout == "packed" else (events, rows)
        if layout != "packed" and positions.shape == (rows,):
            positions = positions.expand(want)
        if tuple(positions.shape) != want:
            raise ValueError(f"positions must be {list(want)}, got {list(positions.shape)}")
        if positions.dtype != torch.int32:
            positions = positions.to(torch.int64)
        positions = positions.to(q.device).contiguous()
    args = (q, k, freqs, cu, positions, layout, bool(interleaved),
            _finite_fp32(magnitude, "magnitude"))
    if seen_by_autograd(q, k):
        return _FlashRotary.apply(*args)
    return _rotate(*args, False)


def flash_rotary(
    q: Tensor,
    k: Optional[Tensor],
    freqs: Tensor,
    positions: Optional[Tensor] = None,
    *,
    layout: str = "bhld",
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Tuple[Tensor, Optional[Tensor]]:
    """Rotate q and k of a padded batch by their positions.

    q: ``[B, H, L, Dh]``, k: ``[B, Hkv, L, Dh]`` or None (``[B, L, heads, Dh]``
    with ``layout='blhd'``; fp32, bf16 or fp16, Dh up to 1024). ``freqs``:
    ``[R/2]`` radians per position for the first R <= Dh channels; the others
    are copied. Channels p and p + R/2 form pair p, or 2p and 2p + 1 when
    ``interleaved``. ``positions``: ``[B, L]`` or ``[L]`` integers, by default
    the row's index; the angle is formed in float64 and off by at most 2e-7
    rad plus ``3 * 2**-53`` of itself (up to positions of about 4e8 the first
    part is the larger one). ``magnitude`` multiplies the rotated channels
    (``rotary_magnitude``). Returns new ``(q, k)`` of the same shapes; every
    row is rotated, padding rows too. Differentiable once in q and k.
    """
    if layout not in ("bhld", "blhd"):
        raise ValueError(f"layout must be 'bhld' or 'blhd', got {layout!r}")
    return _apply(q, k, freqs, None, positions, layout, interleaved, magnitude)


def flash_rotary_varlen(
    q: Tensor,
    k: Optional[Tensor],
    freqs: Tensor,
    cu_seqlens: Optional[Tensor] = None,
    positions: Optional[Tensor] = None,
    *,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Tuple[Tensor, Optional[Tensor]]:
    """Rotate packed q ``[T, H, Dh]`` and k ``[T, Hkv, Dh]`` (or None).

    A row's position is its index in its event (``cu_seqlens``, ``[B+1]``
    ascending offsets; rows of no event are copied unrotated), or
    ``positions`` ``[T]`` when given. The rest as for :func:`flash_rotary`.
    """
    cu = None
    if positions is None:
        if cu_seqlens is None:
            raise ValueError("pass cu_seqlens or positions")
        cu = _integers(cu_seqlens, "cu_seqlens")
        if cu.dim() != 1 or cu.numel() < 1:
            raise ValueError("cu_seqlens must be a [B+1] tensor")
        cu = _int32(cu, 2**31 - 1, q.device)
    return _apply(q, k, freqs, cu, positions, "packed", interleaved, magnitude)
