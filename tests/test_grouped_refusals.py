"""CPU checks of the grouped-head attention and rotary entry points: refusals
before any launch, struct layouts, and the definitions in ``reference``."""

import ctypes
import math
import os
import shutil
import subprocess
import tempfile

import pytest
import torch

import grouped_cases as gc
from flash_spacetime import (_lib, flash_grouped_attention, flash_grouped_attention_varlen,
                             flash_rotary, flash_rotary_varlen, grouped_attention_reference,
                             rotary_frequencies, rotary_magnitude, rotary_reference)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_the_header():
    names = ("FstRows", "FstGroupedProblem", "FstGroupedForwardArgs", "FstGroupedBackwardArgs",
             "FstRotaryArgs")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "flash_spacetime.h"',
             "int main(void) {"]
    for name in names:
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _ in getattr(_lib, name)._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "layout.c"), os.path.join(tmp, "layout")
        open(src, "w").write("\n".join(lines + ["return 0;", "}"]))
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        got = dict(x.split() for x in subprocess.check_output([exe]).decode().split("\n") if x)
    for name in names:
        cls = getattr(_lib, name)
        assert int(got[name]) == ctypes.sizeof(cls)
        for field, _ in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, f"{name}.{field}"


def test_packed_argument_formats_have_the_struct_sizes():
    from flash_spacetime import grouped, rotary
    for fmt, cls in ((grouped._FORWARD, _lib.FstGroupedForwardArgs),
                     (grouped._BACKWARD, _lib.FstGroupedBackwardArgs),
                     (rotary._ROTARY, _lib.FstRotaryArgs)):
        assert fmt.size == ctypes.sizeof(cls)
    # Field by field: distinct values in, the same out of the ctypes mirror.
    a = _lib.FstGroupedForwardArgs.from_buffer_copy(grouped._FORWARD.pack(*range(1, 35)))
    assert [getattr(a.prob, f) for f, _ in a.prob._fields_] == list(range(1, 14))
    assert (a.q.data, a.q.row_stride, a.out_low.event_stride, a.lse) == (14, 17, 31, 34)
    b = _lib.FstGroupedBackwardArgs.from_buffer_copy(grouped._BACKWARD.pack(*range(1, 52)))
    assert (b.dout.data, b.dv.row_stride, b.lse, b.stats) == (34, 49, 50, 51)
    r = _lib.FstRotaryArgs.from_buffer_copy(rotary._ROTARY.pack(*range(1, 33)))
    assert [getattr(r, f) for f, _ in r._fields_[:16]] == list(range(1, 17))
    assert (r.q.data, r.k_out.row_stride) == (17, 32)


def _grouped_args(**kw):
    a = _lib.FstGroupedForwardArgs()
    p = a.prob
    p.dtype, p.packed, p.batch, p.heads, p.kv_heads, p.head_dim = 1, 1, 2, 4, 2, 32
    p.total_rows, p.scale, p.cu_seqlens = 64, 0.5, 256  # never dereferenced
    for key, value in kw.items():
        setattr(p, key, value)
    return a


@pytest.mark.parametrize("change, text", [
    (dict(dtype=3), "dtype"), (dict(kv_heads=3), "multiple"), (dict(kv_heads=0), "sizes"),
    (dict(head_dim=129), "<= 128"), (dict(head_dim=0), "sizes"), (dict(heads=-1), "sizes"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(flags=1), "flags"), (dict(packed=2), "layout"), (dict(cu_seqlens=None), "cu_seqlens"),
    (dict(total_rows=1 << 31), "at most"), (dict(total_rows=-1), "sizes"),
    (dict(packed=0, seqlens=256, max_len=30), "B*L"), (dict(packed=0, max_len=32), "seqlens"),
    (dict(heads=1 << 20, kv_heads=1 << 20, total_rows=1 << 30), "too many"),
    (dict(), "required"),
])
def test_c_abi_refusals(change, text):
    lib = _lib.load()
    a = _grouped_args(**change)
    rc = lib.fst_grouped_forward(ctypes.byref(a), None)
    assert rc in (_lib.FST_ERR_INVALID, _lib.FST_ERR_UNSUPPORTED) and text in _lib.last_error()
    b = _lib.FstGroupedBackwardArgs()
    b.prob = a.prob
    rc = lib.fst_grouped_backward(ctypes.byref(b), None)
    assert rc in (_lib.FST_ERR_INVALID, _lib.FST_ERR_UNSUPPORTED) and text in _lib.last_error()


def test_c_abi_empty_problems_launch_nothing():
    lib = _lib.load()
    before = lib.fst_kernel_launches()
    assert lib.fst_grouped_forward(ctypes.byref(_grouped_args(total_rows=0)), None) == _lib.FST_OK
    a = _lib.FstRotaryArgs()
    a.dtype, a.packed, a.heads, a.head_dim, a.magnitude = 1, 1, 1, 8, 1.0
    assert lib.fst_rotary(ctypes.byref(a), None) == _lib.FST_OK
    assert lib.fst_kernel_launches() == before
    for entry in (lib.fst_grouped_forward, lib.fst_grouped_backward, lib.fst_rotary):
        assert entry(None, None) == _lib.FST_ERR_INVALID


@pytest.mark.parametrize("change, text", [
    (dict(dtype=-1), "dtype"), (dict(pairs=17), "fit"), (dict(pairs=-1), "fit"),
    (dict(head_dim=1025), "1024"), (dict(magnitude=float("nan")), "finite"),
    (dict(packed=3), "layout"), (dict(packed=0, max_len=3), "B*L"), (dict(heads=0), "sizes"),
    (dict(cu_seqlens=None), "positions"), (dict(), "null"),
])
def test_rotary_c_abi_refusals(change, text):
    a = _lib.FstRotaryArgs()
    a.dtype, a.packed, a.batch, a.heads, a.head_dim, a.pairs = 1, 1, 2, 4, 32, 16
    a.magnitude, a.total_rows, a.cu_seqlens = 1.0, 64, 256
    for key, value in change.items():
        setattr(a, key, value)
    rc = _lib.load().fst_rotary(ctypes.byref(a), None)
    assert rc in (_lib.FST_ERR_INVALID, _lib.FST_ERR_UNSUPPORTED) and text in _lib.last_error()


def _meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_python_refusals():
    q, k = _meta(8, 4, 32), _meta(8, 2, 32)
    cu = torch.tensor([0, 8])
    with pytest.raises(ValueError, match="CUDA"):
        flash_grouped_attention_varlen(q, k, k, cu)
    with pytest.raises(ValueError, match="CUDA"):
        flash_grouped_attention(_meta(1, 4, 8, 32), _meta(1, 2, 8, 32), _meta(1, 2, 8, 32))
    with pytest.raises(ValueError, match="dtype"):
        flash_grouped_attention_varlen(q.double(), k.double(), k.double(), cu)
    with pytest.raises(ValueError, match="CUDA"):
        flash_rotary_varlen(q, k, rotary_frequencies(32), cu)
    with pytest.raises(ValueError, match="cu_seqlens or positions"):
        flash_rotary_varlen(q, k, rotary_frequencies(32))
    with pytest.raises(ValueError, match="layout"):
        flash_rotary(q, k, rotary_frequencies(32), layout="packed")
    with pytest.raises(ValueError, match="integers"):
        flash_rotary_varlen(q, k, rotary_frequencies(32), torch.tensor([0.0, 8.0]))


def test_reference_matches_the_case_results():
    events = gc.make_case([9, 0, 5], 4, 2, 8, torch.float32, True)
    q, k, v = (gc.pad(events, x, 9, "bhld").double() for x in "qkv")
    out = grouped_attention_reference(q, k, v, torch.tensor([9, 0, 5]))
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    for b, n in ((0, 9), (2, 5)):
        assert (out[b, :, :n] - events[b]["out"]).abs().max() < 1e-12
        assert torch.equal(out[b, :, n:], torch.zeros_like(out[b, :, n:]))


def test_rotary_frequencies():
    f = rotary_frequencies(8)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert torch.allclose(rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    base = rotary_frequencies(8, scaling="base", factor=4.0)
    assert base[0] == 1.0 and math.isclose(base[-1], f[-1] / 4, rel_tol=1e-12)
    parts = rotary_frequencies(64, scaling="parts", factor=8.0)
    plain = rotary_frequencies(64)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    assert torch.allclose(parts[turns <= 1], plain[turns <= 1] / 8)
    assert (parts.diff() < 0).all()
    assert rotary_magnitude(1.0) == 1.0 and math.isclose(rotary_magnitude(math.e), 1.1)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=4, scaling="x"),
                dict(rotary_dim=4, factor=0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_reference_turns_pairs(interleaved):
    x = torch.tensor([1.0, 0.0, 7.0]) if interleaved else torch.tensor([1.0, 0.0, 7.0])
    got = rotary_reference(x, torch.tensor([math.pi / 2], dtype=torch.float64), torch.tensor(1),
                           interleaved)
    assert torch.allclose(got, torch.tensor([0.0, 1.0, 7.0]), atol=1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_reference_pairs_channels(interleaved):
    # Three pairs turned by 90, 180 and 0 degrees, a channel behind them; by
    # halves (0, 3) (1, 4) (2, 5), or neighbours.
    freqs = torch.tensor([math.pi / 2, math.pi, 0.0], dtype=torch.float64)
    x = torch.arange(1.0, 8.0, dtype=torch.float64)
    want = ([-2.0, 1.0, -3.0, -4.0, 5.0, 6.0, 7.0] if interleaved
            else [-4.0, -2.0, 3.0, 1.0, -5.0, 6.0, 7.0])
    got = rotary_reference(x, freqs, torch.tensor(1), interleaved)
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), atol=1e-12)
    doubled = rotary_reference(x, freqs, torch.tensor(1), interleaved, magnitude=2.0)
    assert torch.allclose(doubled[:6], 2 * got[:6]) and doubled[6] == 7.0


def _fill(a, size):
    """Every pointer of an argument struct set to an address that is aligned to
    ``size`` bytes; none is ever read."""
    address = 4096 + size
    for name, kind in a._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, address)
        elif kind is _lib.FstRows:
            getattr(a, name).data = address
    return a


@pytest.mark.parametrize("dtype, size", [(_lib.FST_F32, 4), (_lib.FST_BF16, 2), (_lib.FST_F16, 2)])
def test_misaligned_pointers_are_refused_before_a_launch(dtype, size):
    lib = _lib.load()
    before = lib.fst_kernel_launches()

    def refused(entry, a):
        assert entry(ctypes.byref(a), None) == _lib.FST_ERR_INVALID
        assert "aligned" in _lib.last_error()

    for entry, cls, names in (
            (lib.fst_grouped_forward, _lib.FstGroupedForwardArgs,
             ("q", "k", "v", "out", "out_low", "lse")),
            (lib.fst_grouped_backward, _lib.FstGroupedBackwardArgs,
             ("q", "k", "v", "out", "out_low", "dout", "dq", "dk", "dv", "lse", "stats"))):
        for name in names:
            a = _fill(cls(), 8)
            a.prob = _grouped_args(dtype=dtype).prob
            if isinstance(getattr(a, name), _lib.FstRows):
                getattr(a, name).data += size // 2
            else:
                setattr(a, name, getattr(a, name) + 2)
            refused(entry, a)
        a = _fill(cls(), 8)
        a.prob = _grouped_args(dtype=dtype, cu_seqlens=258).prob
        refused(entry, a)
    for name, off in (("q", size // 2), ("k_out", size // 2), ("freqs", 4), ("cu_seqlens", 2),
                      ("positions", 4)):
        a = _fill(_lib.FstRotaryArgs(), 8)
        a.dtype, a.packed, a.batch, a.heads, a.kv_heads, a.head_dim, a.pairs = dtype, 1, 2, 4, 2, 32, 16
        a.magnitude, a.total_rows, a.positions_64 = 1.0, 64, 1
        if isinstance(getattr(a, name), _lib.FstRows):
            getattr(a, name).data += off
        else:
            setattr(a, name, getattr(a, name) + off)
        refused(lib.fst_rotary, a)
    assert lib.fst_kernel_launches() == before
