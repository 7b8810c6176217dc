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
