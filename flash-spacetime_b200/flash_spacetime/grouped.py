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
* with gradients, a 16-bit forward also keeps what rounding its output left
  over, so that the backward's row sums ``D = dO . out`` are those of the
  unrounded output: dq and dk would otherwise carry its rounding, times any
  offset that the values share (an offset of the keys stays out of dq as well);
* a row that sees one key (the row of an event of one, row 0 of a causal event)
  has a dq, and a share in dk, of exactly 0;
* fp16 gradients keep their small values whatever the gradient's scale: dS
  carries powers of two taken from the event's largest finite values;
* calls without a gradient launch directly, unless a trace is being recorded or
  a forward-mode level or ``torch.func`` transform is active, which the autograd
  node runs or refuses;
* inputs are read in place whatever their strides, as long as the channels of
  a head are adjacent: slices of a fused projection need no copy;
* forward and backward may be captured into CUDA graphs (lengths on the device;
  a list is copied, which a capture refuses). PyTorch's own rule holds for
  ``.backward()`` in a capture: no eager graph of the same leaves may be alive.
"""

import struct
from typing import Any, Callable, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPES, _padded_lengths, _timed_call

# The argument structs of the C ABI, packed in one go: filling ctypes
# structures field by field would take longer than a small call's kernels.
# FstRows is (data, event, head, row stride).
_PROBLEM = "8iqfi2Q"
_ROWS = "Q3q"
_FORWARD = struct.Struct("@" + _PROBLEM + 5 * _ROWS + "Q")
_BACKWARD = struct.Struct("@" + _PROBLEM + 9 * _ROWS + "2Q")
_NO_ROWS = (0, 0, 0, 0)
_CONTIGUOUS = torch.contiguous_format

Sizes = Tuple[int, int, int, int]


def _in_place(t: Tensor) -> Tensor:
    """``t`` itself where the kernels can read it in place, else a copy.

    A head's channels must be adjacent, and no stride 0 (an expanded tensor).
    For 16-bit tensors whose head is a whole number of 16-byte vectors, rows
    off the 16-byte grid are copied too: the tensor-core kernels need it.
    """
    aligned = t.data_ptr() % 16 == 0
    if aligned and t.is_contiguous():
        return t
    if t.element_size() == 2 and t.shape[-1] % 8 == 0:
        aligned = aligned and all(
            s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
    else:
        aligned = True
    strided = all(s > 0 for s, n in zip(t.stride(), t.shape) if n > 1)
    if aligned and strided and (t.stride(-1) == 1 or t.shape[-1] == 1):
        return t
    return t.clone(memory_format=_CONTIGUOUS)


def _rows(t: Tensor, layout: str) -> Tuple[int, int, int, int]:
    s = t.stride()
    if layout == "packed":
        return t.data_ptr(), 0, s[1], s[0]
    if layout == "bhld":
        return t.data_ptr(), s[0], s[1], s[2]
    return t.data_ptr(), s[0], s[2], s[1]


def _integers(t: Tensor, what: str) -> Tensor:
    if not isinstance(t, Tensor):
        raise ValueError(f"{what} must be a tensor of integers, got {type(t).__name__}")
    if t.dtype == torch.bool or t.dtype.is_floating_point or t.dtype.is_complex:
        raise ValueError(f"{what} must be integers, got {t.dtype}")
    return t


def _int32(t: Tensor, most: int, device: torch.device) -> Tensor:
    """``t`` as int32 on ``device``; wider types are clamped to [0, most], so
    that nothing wraps (the kernels clamp int32 themselves)."""
    if t.dtype == torch.uint64:  # above 2^63 - 1 as an int64: negative
        t = t.to(torch.int64)
        t = torch.where(t < 0, torch.full_like(t, most), t)
    if t.dtype in (torch.int64, torch.uint32):
        t = t.to(torch.int64).clamp(0, most)
    return t.to(device=device, dtype=torch.int32).contiguous()


def _finite_fp32(x: float, what: str) -> float:
    x = float(x)
    if not abs(x) <= torch.finfo(torch.float32).max:
        raise ValueError(f"{what} must be finite in fp32, got {x}")
    return x


def _bool_mask(mask: Any, shape: Tuple[int, int], validate: bool) -> Any:
    """A 2-D padding mask as bool (True: padding); anything else as it is. A float
    mask marks padding with -inf or its type's lowest value, valid rows with 0."""
    if not isinstance(mask, Tensor) or mask.dim() != 2:
        return mask
    if mask.shape != shape:
        raise ValueError(f"a padding mask must be [B, L] = [{shape[0]}, {shape[1]}], got "
                         f"{tuple(mask.shape)}")
    if mask.dtype == torch.bool:
        return mask
    if not mask.dtype.is_floating_point:
        raise ValueError(f"a padding mask must be bool or float, got {mask.dtype}")
    padding = mask <= torch.finfo(mask.dtype).min
    if validate and bool((~padding & (mask != 0)).any()):
        raise ValueError("a float padding mask must be 0 (valid) or -inf or its type's lowest "
                         "value (padding) everywhere")
    return padding


def _shape(t: Tensor, layout: str, what: str) -> Sizes:
    """(events, rows per event or in all, heads, Dh) of a tensor."""
    shape = t.shape
    if layout == "packed":
        if len(shape) != 3:
            raise ValueError(f"varlen {what} must be [T, H, D], got {tuple(shape)}")
        return 0, shape[0], shape[1], shape[2]
    if layout not in ("bhld", "blhd"):
        raise ValueError(f"layout must be 'bhld' or 'blhd', got {layout!r}")
    if len(shape) != 4:
        raise ValueError(f"{what} must be [B, H, L, D] (or [B, L, H, D] with layout='blhd'), "
                         f"got {tuple(shape)}")
    if layout == "blhd":
        return shape[0], shape[1], shape[2], shape[3]
    return shape[0], shape[2], shape[1], shape[3]


def _check_tensor(t: Tensor, q: Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError("flash_spacetime runs on CUDA tensors only")
    if t.device != q.device:
        raise ValueError(f"{what} is on {t.device}, q on {q.device}")
    if t.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")


def _on_device(index: int, run: Callable[[int], Any]) -> Any:
    """``run(stream)`` with the device current and its current stream."""
    if torch.cuda.current_device() == index:
        return run(torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return run(torch._C._cuda_getCurrentRawStream(index))


def _call(name: str, args: bytes, device: torch.device) -> None:
    entry = getattr(_lib.load(), name)
    rc = _on_device(device.index,
                    lambda stream: _timed_call(name, entry, (args, stream), device))
    if rc:
        _lib.check(rc, name)


def _problem(q: Tensor, kv_heads: int, layout: str, lens: Tensor, scale: float,
             causal: bool) -> Tuple[Any, ...]:
    events, rows, heads, dim = _shape(q, layout, "q")
    dtype = _DTYPES[q.dtype]
    if layout == "packed":
        return (dtype, 1, lens.shape[0] - 1, heads, kv_heads, 0, dim, causal, rows, scale, 0,
                0, lens.data_ptr())
    return (dtype, 0, events, heads, kv_heads, rows, dim, causal, events * rows, scale, 0,
            lens.data_ptr(), 0)


def _forward(q: Tensor, k: Tensor, v: Tensor, lens: Tensor, layout: str, scale: float,
             causal: bool, keep_low: bool = False) -> Tuple[Any, ...]:
    """One ``fst_grouped_forward`` call: out, lse, q, k, v as read, and with
    ``keep_low`` what rounding a 16-bit out left over (else None)."""
    q, k, v = _in_place(q), _in_place(k), _in_place(v)
    events, rows, heads, _ = _shape(q, layout, "q")
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    low = torch.empty_like(out) if keep_low and q.element_size() == 2 else None
    shape = (heads, rows) if layout == "packed" else (events, heads, rows)
    lse = q.new_empty(shape, dtype=torch.float32)
    args = _FORWARD.pack(
        *_problem(q, _shape(k, layout, "k")[2], layout, lens, scale, causal), *_rows(q, layout),
        *_rows(k, layout), *_rows(v, layout), *_rows(out, layout),
        *(_NO_ROWS if low is None else _rows(low, layout)), lse.data_ptr())
    _call("fst_grouped_forward", args, q.device)
    return out, lse, q, k, v, low


class _FlashGroupedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Tensor, v: Tensor, lens: Tensor, layout: str,
                scale: float, causal: bool) -> Tensor:  # type: ignore[override]
        out, lse, q, k, v, low = _forward(q, k, v, lens, layout, scale, causal, True)
        ctx.save_for_backward(q, k, v, out, low, lse, lens)
        ctx.layout, ctx.scale, ctx.causal = layout, scale, causal
        return out

    @staticmethod
    def backward(ctx: Any, grad_out: Tensor) -> Tuple[Optional[Tensor], ...]:  # type: ignore[override]
        return once(_backward)(ctx, grad_out)


def once(backward: Callable[..., Any]) -> Callable[..., Any]:
    """``backward``, refusing to be differentiated again. Only a backward pass
    that builds a graph itself can be, and only it pays for the refusal."""
    return once_differentiable(backward) if torch.is_grad_enabled() else backward


def seen_by_autograd(*tensors: Optional[Tensor]) -> bool:
    """Whether a call must go through its ``autograd.Function``.

    For a gradient, and wherever something else follows the call and would not
    see a bare launch: a trace would record the empty output alone, and
    forward-mode derivatives or ``torch.func`` transforms would be dropped
    where the Function refuses them. Other calls launch directly.
    """
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return (forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None
            or torch._C._functorch.peek_interpreter_stack() is not None)


def _backward(ctx: Any, grad_out: Tensor) -> Tuple[Optional[Tensor], ...]:
    """One ``fst_grouped_backward`` call."""
    q, k, v, out, low, lse, lens = ctx.saved_tensors
    layout = ctx.layout
    dout = _in_place(grad_out)
    dq, dk, dv = (torch.empty_like(t, memory_format=_CONTIGUOUS) for t in (q, k, v))
    kv_heads, heads = _shape(k, layout, "k")[2], _shape(q, layout, "q")[2]
    stats = lse.new_empty((2 * heads + kv_heads) * (lse.numel() // heads))
    args = _BACKWARD.pack(
        *_problem(q, kv_heads, layout, lens, ctx.scale, ctx.causal),
        *_rows(q, layout), *_rows(k, layout), *_rows(v, layout), *_rows(out, layout),
        *(_NO_ROWS if low is None else _rows(low, layout)), *_rows(dout, layout),
        *_rows(dq, layout), *_rows(dk, layout), *_rows(dv, layout), lse.data_ptr(), stats.data_ptr())
    _call("fst_grouped_backward", args, q.device)
    need = ctx.needs_input_grad
    return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
            None, None, None, None)


def _check_heads(q: Tensor, k: Tensor, v: Tensor, layout: str) -> Sizes:
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    _check_tensor(q, q, "q")
    _check_tensor(k, q, "k")
    _check_tensor(v, q, "v")
    sizes = events, rows, heads, dim = _shape(q, layout, "q")
    k_events, k_rows, kv_heads, k_dim = _shape(k, layout, "k")
    if (k_events, k_rows, k_dim) != (events, rows, dim) or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have q's events, rows "
                         f"and Dh, q is {tuple(q.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"the heads of q ({heads}) must be a multiple of those of k ({kv_heads})")
    if not 1 <= dim <= 128:
        raise ValueError(f"Dh (={dim}) must be 1 to 128")
    if max(1, events) * rows >= 2**31 - 255:
        raise ValueError(f"q has {max(1, events) * rows} rows, at most {2**31 - 256} are supported")
    return sizes


def _apply(q: Tensor, k: Tensor, v: Tensor, lens: Tensor, layout: str, scale: Optional[float],
           causal: bool) -> Tensor:
    args = (q, k, v, lens, layout,
            _finite_fp32(q.shape[-1]**-0.5 if scale is None else scale, "scale"), bool(causal))
    if seen_by_autograd(q, k, v):
        return _FlashGroupedAttention.apply(*args)
    return _forward(*args)[0]


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
    :func:`flash_spacetime_attention`, whose float form may also mark padding
    with its type's lowest value; None means that every row is valid. Integer
    masks are refused, and with ``validate_mask`` other float values.
    ``scale`` multiplies the logits (default ``Dh**-0.5``). With ``causal``
    row i sees the rows j <= i of its event, else all of them.

    Returns q's shape and dtype, padding rows exactly 0. Values in an event's
    valid rows are expected to be finite: an infinity or NaN there may also
    reach the rows of its event that do not see it. Padding rows may hold
    anything.
    """
    events, rows, _, _ = _check_heads(q, k, v, layout)
    if isinstance(seqlens, Tensor) and seqlens.dim() == 1:
        _integers(seqlens, "seqlens")
    seqlens, key_padding_mask = (_bool_mask(m, (events, rows), validate_mask)
                                 for m in (seqlens, key_padding_mask))
    lens, _ = _padded_lengths(seqlens, key_padding_mask, events, rows, q.device, validate_mask,
                              None)
    if not isinstance(lens, Tensor):
        lens = torch.as_tensor(lens)
        lens = lens if lens.numel() else lens.to(torch.int64)  # an empty list has no type
    lens = _int32(_integers(lens, "seqlens"), rows, q.device)
    if lens.shape != (events,):
        raise ValueError(f"seqlens must be [B] = [{events}], got {tuple(lens.shape)}")
    return _apply(q, k, v, lens, layout, scale, causal)


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
    cu = _int32(_integers(cu_seqlens, "cu_seqlens"), q.shape[0], q.device)
    return _apply(q, k, v, cu, "packed", scale, causal)
