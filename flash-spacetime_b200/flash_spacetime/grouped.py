"""Grouped-head attention: the blocks of a model that have no pair term.

``flash_grouped_attention`` (padded) and ``flash_grouped_attention_varlen``
(packed) take the layouts, lengths and masks of the spacetime ops of ``ops``;
k and v may have fewer heads than q, and the attention may be causal (the
default) or see the whole event. Behind them one ``torch.autograd.Function``
calls ``fst_grouped_forward`` / ``fst_grouped_backward``; there is no other
code path.

Conventions:

* q head ``h`` reads k / v head ``h // (H / Hkv)``; dk and dv are summed over
  the heads that share them;
* rows of no event (padding; packed rows outside the offsets) are never read,
  and are exactly 0 in the output and in every gradient;
* softmax statistics and sums are fp32; results are bitwise deterministic run
  to run (no atomics);
* inputs are read in place whatever their strides, as long as the channels of
  a head are adjacent: slices of a fused projection need no copy.
"""

import ctypes
from typing import Any, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPES, _padded_lengths, _ptr, _stream, _timed_call


def _in_place(t: Tensor) -> Tensor:
    """``t`` itself where the kernels can read it in place, else a copy.

    A head's channels must be adjacent, and no stride 0 (an expanded tensor).
    For 16-bit tensors whose head is a whole number of 16-byte vectors, rows
    off the 16-byte grid are copied too: the tensor-core kernels need it.
    """
    aligned = True
    if t.element_size() == 2 and t.shape[-1] % 8 == 0:
        aligned = t.data_ptr() % 16 == 0 and all(
            s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
    strided = all(s > 0 for s, n in zip(t.stride(), t.shape) if n > 1)
    if aligned and strided and (t.stride(-1) == 1 or t.shape[-1] == 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _rows(t: Optional[Tensor], layout: str) -> _lib.FstRows:
    r = _lib.FstRows()
    if t is None:
        return r
    r.data = _ptr(t)
    if layout == "packed":
        r.row_stride, r.head_stride = t.stride(0), t.stride(1)
    elif layout == "bhld":
        r.event_stride, r.head_stride, r.row_stride = t.stride(0), t.stride(1), t.stride(2)
    else:
        r.event_stride, r.row_stride, r.head_stride = t.stride(0), t.stride(1), t.stride(2)
    return r


def _integers(t: Tensor, what: str) -> Tensor:
    if t.dtype == torch.bool or t.dtype.is_floating_point or t.dtype.is_complex:
        raise ValueError(f"{what} must be integers, got {t.dtype}")
    return t


def _shape(t: Tensor, layout: str, what: str) -> Tuple[int, int, int, int]:
    """(events, rows per event or in all, heads, Dh) of a tensor."""
    if layout == "packed":
        if t.dim() != 3:
            raise ValueError(f"varlen {what} must be [T, H, D], got {tuple(t.shape)}")
        return 0, t.shape[0], t.shape[1], t.shape[2]
    if layout not in ("bhld", "blhd"):
        raise ValueError(f"layout must be 'bhld' or 'blhd', got {layout!r}")
    if t.dim() != 4:
        raise ValueError(f"{what} must be [B, H, L, D] (or [B, L, H, D] with layout='blhd'), "
                         f"got {tuple(t.shape)}")
    if layout == "blhd":
        return t.shape[0], t.shape[1], t.shape[2], t.shape[3]
    return t.shape[0], t.shape[2], t.shape[1], t.shape[3]


def _check_tensor(t: Tensor, q: Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError("flash_spacetime runs on CUDA tensors only")
    if t.device != q.device:
        raise ValueError(f"{what} is on {t.device}, q on {q.device}")
    if t.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")


def _problem(q: Tensor, k: Tensor, layout: str, lens: Tensor, scale: float,
             causal: bool) -> _lib.FstGroupedProblem:
    events, rows, heads, dim = _shape(q, layout, "q")
    p = _lib.FstGroupedProblem()
    p.dtype = _DTYPES[q.dtype]
    p.packed = int(layout == "packed")
    p.heads, p.kv_heads = heads, _shape(k, layout, "k")[2]
    p.head_dim, p.causal, p.scale = dim, int(causal), scale
    if p.packed:
        p.batch, p.total_rows, p.cu_seqlens = lens.numel() - 1, rows, _ptr(lens)
    else:
        p.batch, p.max_len, p.total_rows, p.seqlens = events, rows, events * rows, _ptr(lens)
    return p


def _lse_shape(q: Tensor, layout: str) -> Tuple[int, ...]:
    events, rows, heads, _ = _shape(q, layout, "q")
    return (heads, rows) if layout == "packed" else (events, heads, rows)


class _FlashGroupedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Tensor, v: Tensor, lens: Tensor, layout: str,
                scale: float, causal: bool) -> Tensor:  # type: ignore[override]
        lib = _lib.load()
        qc, kc, vc = _in_place(q), _in_place(k), _in_place(v)
        with torch.cuda.device(q.device):
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            lse = torch.empty(_lse_shape(q, layout), dtype=torch.float32, device=q.device)
            a = _lib.FstGroupedForwardArgs()
            a.prob = _problem(qc, kc, layout, lens, scale, causal)
            a.q, a.k, a.v, a.out = (_rows(t, layout) for t in (qc, kc, vc, out))
            a.lse = _ptr(lse)
            rc = _timed_call("fst_grouped_forward", lib.fst_grouped_forward,
                             (ctypes.byref(a), _stream(q.device)), q.device)
        _lib.check(rc, "fst_grouped_forward")
        ctx.save_for_backward(qc, kc, vc, out, lse, lens)
        ctx.layout, ctx.scale, ctx.causal = layout, scale, causal
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_out: Tensor) -> Tuple[Optional[Tensor], ...]:  # type: ignore[override]
        q, k, v, out, lse, lens = ctx.saved_tensors
        lib, layout = _lib.load(), ctx.layout
        with torch.cuda.device(q.device):
            dout = _in_place(grad_out)
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device)
                          for t in (q, k, v))
            stats = torch.empty(2 * lse.numel(), dtype=torch.float32, device=q.device)
            a = _lib.FstGroupedBackwardArgs()
            a.prob = _problem(q, k, layout, lens, ctx.scale, ctx.causal)
            a.q, a.k, a.v, a.out, a.dout = (_rows(t, layout) for t in (q, k, v, out, dout))
            a.dq, a.dk, a.dv = (_rows(t, layout) for t in (dq, dk, dv))
            a.lse, a.stats = _ptr(lse), _ptr(stats)
            rc = _timed_call("fst_grouped_backward", lib.fst_grouped_backward,
                             (ctypes.byref(a), _stream(q.device)), q.device)
        _lib.check(rc, "fst_grouped_backward")
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
                None, None, None, None)


def _check_heads(q: Tensor, k: Tensor, v: Tensor, layout: str) -> None:
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_tensor(t, q, name)
    events, rows, heads, dim = _shape(q, layout, "q")
    if _shape(k, layout, "k")[:2] != (events, rows) or k.shape[-1] != dim or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have q's events, rows "
                         f"and Dh, q is {tuple(q.shape)}")
    kv_heads = _shape(k, layout, "k")[2]
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"the heads of q ({heads}) must be a multiple of those of k ({kv_heads})")
    if not 1 <= dim <= 128:
        raise ValueError(f"Dh (={dim}) must be 1 to 128")


def flash_grouped_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    seqlens: Optional[Tensor] = None,
    scale: Optional[float] = None,
    *,
    causal: bool = True,
    key_padding_mask: Optional[Tensor] = None,
    layout: str = "bhld",
    validate_mask: bool = True,
) -> Tensor:
    """Attention without the pair term on a padded batch.

    q: ``[B, H, L, Dh]``; k, v: ``[B, Hkv, L, Dh]`` with Hkv a divisor of H and
    Dh at most 128 (fp32, bf16 or fp16); with ``layout='blhd'`` all are
    ``[B, L, heads, Dh]``. ``seqlens`` is the ``[B]`` valid prefix lengths
    (on any device, or a list; clamped to ``[0, L]``) or a ``[B, L]`` padding mask, as for
    :func:`flash_spacetime_attention`; None means that every row is valid.
    ``scale`` multiplies the logits (default ``Dh**-0.5``). With ``causal``
    row i sees the rows j <= i of its event, else all of them.

    Returns q's shape and dtype, padding rows exactly 0. Values in an event's
    valid rows are expected to be finite: an infinity or NaN there may also
    reach the rows of its event that do not see it. Padding rows may hold
    anything.
    """
    _check_heads(q, k, v, layout)
    events, rows, _, _ = _shape(q, layout, "q")
    if isinstance(seqlens, Tensor) and seqlens.dim() == 1:
        _integers(seqlens, "seqlens")
    lens, _ = _padded_lengths(seqlens, key_padding_mask, events, rows, q.device, validate_mask,
                              None)
    lens = _integers(torch.as_tensor(lens), "seqlens")
    if lens.dtype == torch.int64:  # must not wrap into 32 bits; the kernels clamp the rest
        lens = lens.clamp(0, rows)
    lens = lens.to(device=q.device, dtype=torch.int32).contiguous()
    if lens.shape != (events,):
        raise ValueError(f"seqlens must be [B] = [{events}], got {tuple(lens.shape)}")
    return _FlashGroupedAttention.apply(q, k, v, lens, layout,
                                        float(q.shape[-1]**-0.5 if scale is None else scale),
                                        bool(causal))


def flash_grouped_attention_varlen(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    cu_seqlens: Tensor,
    scale: Optional[float] = None,
    *,
    causal: bool = True,
) -> Tensor:
    """Attention without the pair term on packed events.

    q: ``[T, H, Dh]``; k, v: ``[T, Hkv, Dh]``; ``cu_seqlens``: ``[B+1]``
    ascending row offsets in ``[0, T]`` (offsets outside are clamped; they
    need not start at 0 or end at T: rows of no event are 0 in the output).
    The rest as for :func:`flash_grouped_attention`. No host synchronisation
    happens.
    """
    _check_heads(q, k, v, "packed")
    if not isinstance(cu_seqlens, Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a [B+1] tensor")
    cu = _integers(cu_seqlens, "cu_seqlens")
    if cu.dtype == torch.int64:
        cu = cu.clamp(0, q.shape[0])
    cu = cu.to(device=q.device, dtype=torch.int32).contiguous()
    return _FlashGroupedAttention.apply(q, k, v, cu, "packed",
                                        float(q.shape[-1]**-0.5 if scale is None else scale),
                                        bool(causal))
