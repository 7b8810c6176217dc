"""Lengths, masks, offsets and scalars of the grouped-head attention and rotary
calls, on the CPU: the launch is replaced by one that records its arguments."""

import ctypes

import pytest
import torch

from flash_spacetime import (_lib, flash_grouped_attention, flash_grouped_attention_varlen,
                             flash_rotary, flash_rotary_varlen, grouped, rotary)

FREQS = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64)


def _ints(address, count, kind=ctypes.c_int32):
    return list((kind * count).from_address(address)) if count else []


@pytest.fixture
def seen(monkeypatch):
    """What each launch was given."""
    calls = []

    def call(name, args, device):
        if name == "fst_rotary":
            a = _lib.FstRotaryArgs.from_buffer_copy(args)
            cu = _ints(a.cu_seqlens, a.batch + 1) if a.cu_seqlens else None
            kind = ctypes.c_int64 if a.positions_64 else ctypes.c_int32
            pos = _ints(a.positions, a.total_rows, kind) if a.positions else None
            calls.append(cu if pos is None else pos)
        else:
            p = _lib.FstGroupedForwardArgs.from_buffer_copy(args).prob
            calls.append(_ints(p.cu_seqlens, p.batch + 1) if p.packed
                         else _ints(p.seqlens, p.batch))

    for module in (grouped, rotary):
        monkeypatch.setattr(module, "_call", call)
        monkeypatch.setattr(module, "_check_tensor", lambda *_: None)
    return calls


def _padded(events, rows=6):
    return torch.zeros(events, 4, rows, 8), torch.zeros(events, 2, rows, 8)


def test_length_forms(seen):
    q, k = _padded(3)
    forms = [[6, 2, 0], (6, 2, 0), torch.tensor([6, 2, 0]), torch.tensor([9, 2, -4]),
             torch.tensor([6, 2, 0], dtype=torch.uint8),
             torch.tensor([2**32 - 1, 2, 0], dtype=torch.uint32),
             torch.tensor([2**64 - 1, 2, 0], dtype=torch.uint64), [2**40, 2, -(2**40)]]
    for form in forms:
        flash_grouped_attention(q, k, k, form)
    assert all(x == [6, 2, 0] for x in seen) and len(seen) == len(forms)


def test_a_batch_of_no_events(seen):
    q, k = _padded(0)
    for form in ([], torch.zeros(0, dtype=torch.int32), None, torch.zeros(0, 6, dtype=torch.bool)):
        assert flash_grouped_attention(q, k, k, form).shape == q.shape
    assert seen == [[]] * 4


@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.bfloat16, torch.float16,
                                   torch.float64])
@pytest.mark.parametrize("how", ["seqlens", "key_padding_mask"])
def test_masks(seen, dtype, how):
    q, k = _padded(3)
    padding = torch.arange(6)[None, :] >= torch.tensor([6, 2, 0])[:, None]
    marks = [1.0] if dtype == torch.bool else [float("-inf"), torch.finfo(dtype).min]
    for mark in marks:
        mask = torch.zeros(3, 6).double().masked_fill(padding, mark).to(dtype)
        for validate in (True, False):
            flash_grouped_attention(q, k, k, **{how: mask}, validate_mask=validate)
    assert len(seen) == 2 * len(marks) and all(x == [6, 2, 0] for x in seen)


def test_masks_that_are_refused(seen):
    q, k = _padded(3)
    ones = torch.ones(3, 6)
    for mask, text in ((ones.long(), "bool or float"), (ones.to(torch.uint8), "bool or float"),
                       (ones, "lowest"), (-1e4 * ones, "lowest"),
                       (float("nan") * ones, "lowest"), (ones[:, :5].bool(), "mask")):
        for how in ("seqlens", "key_padding_mask"):
            with pytest.raises(ValueError, match=text):
                flash_grouped_attention(q, k, k, **{how: mask})
    assert not seen


def test_offsets(seen):
    q, k = torch.zeros(6, 4, 8), torch.zeros(6, 2, 8)
    top = {torch.int32: 2**31 - 1, torch.int64: 2**40, torch.uint32: 2**32 - 1,
           torch.uint64: 2**64 - 1}
    for dtype, far in top.items():
        cu = torch.tensor([0, 4, far], dtype=dtype)
        flash_grouped_attention_varlen(q, k, k, cu)
        flash_rotary_varlen(q, k, FREQS, cu)
    assert all(x[:2] == [0, 4] and x[2] >= 6 for x in seen) and len(seen) == 8
    for bad in ([0, 6], None, torch.tensor(6), torch.tensor([0.0, 6.0]), torch.zeros(0).long()):
        with pytest.raises(ValueError):
            flash_grouped_attention_varlen(q, k, k, bad)
        with pytest.raises(ValueError):
            flash_rotary_varlen(q, k, FREQS, bad)


def test_positions_of_unsigned_types(seen):
    q, k = torch.zeros(2, 4, 8), torch.zeros(2, 2, 8)
    for dtype, far in ((torch.uint8, 255), (torch.int16, -7), (torch.uint32, 2**32 - 1),
                       (torch.int64, 2**40), (torch.int32, -1)):
        flash_rotary_varlen(q, k, FREQS, positions=torch.tensor([3, far], dtype=dtype))
        assert seen[-1] == [3, far]
    for bad in ([3, 4], torch.tensor([3.0, 4.0])):
        with pytest.raises(ValueError):
            flash_rotary_varlen(q, k, FREQS, positions=bad)


@pytest.mark.parametrize("value", [1e39, -1e39, float("inf"), float("nan")])
def test_scalars_past_fp32_are_refused(seen, value):
    q, k = _padded(1)
    with pytest.raises(ValueError, match="finite"):
        flash_grouped_attention(q, k, k, scale=value)
    with pytest.raises(ValueError, match="finite"):
        flash_rotary(q, k, FREQS, magnitude=value)
    with pytest.raises(ValueError, match="freqs"):
        flash_rotary(q, k, [1.0, 0.1])
    assert not seen


def test_row_counts_past_32_bits_are_refused(seen):
    q = torch.zeros(1).expand(2, 1, 2**30, 8)
    with pytest.raises(ValueError, match="rows"):
        flash_grouped_attention(q, q, q)
    q = torch.zeros(1).expand(1, 1, 2**31, 8)
    with pytest.raises(ValueError, match="rows"):
        flash_rotary(q, q, FREQS)
    assert not seen
