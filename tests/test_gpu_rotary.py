"""Rotary positions against the float64 definition.

A result is x cos - y sin in fp32 from cos and sin that are off by at most
2^-22 (the reduced angle's rounding, 2^-25 turns = 1.9e-7 rad, and two ulp of
sincospi, times the magnitude m), rounded once: the bound is
u |ref| + 2^-21 m (|x| + |y|), u half a step of the type.
"""

import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime import (flash_rotary, flash_rotary_varlen, rotary_frequencies,
                                 rotary_magnitude, rotary_reference)

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _check(got, x, freqs, pos, interleaved, mag):
    x, got = x.detach().cpu(), got.detach().cpu()
    pos = pos.cpu()
    assert got.dtype == x.dtype and got.shape == x.shape
    ref = rotary_reference(x.double(), freqs, pos, interleaved, mag)
    rot = 2 * freqs.numel()
    part = torch.zeros_like(ref)
    head = x[..., :rot].double().abs()
    if interleaved:
        part[..., :rot] = head.unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1)
    else:
        half = head.unflatten(-1, (2, -1)).sum(-2)
        part[..., :rot] = torch.cat((half, half), -1)
    bound = torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0**-21 * mag * part
    bound += torch.finfo(x.dtype).tiny
    worst = ((got.double() - ref).abs() / bound).max().item() if x.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.2f} times its bound"
    assert torch.equal(got[..., rot:], x[..., rot:])


def _event_positions(lens):
    return torch.cat([torch.arange(n) for n in lens])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, rot", [(32, 32), (32, 16), (64, 24), (128, 128), (48, 20), (80, 40),
                                      (7, 6), (33, 2), (256, 256), (16, 0), (2, 2), (1024, 1024)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_packed(dtype, dim, rot, interleaved):
    lens = [5, 1, 0, 70, 33]
    gen = torch.Generator(device="cuda").manual_seed(dim)
    t = [torch.randn(sum(lens), h, dim, device="cuda", generator=gen).to(dtype)
         for h in (3, 1, 3, 1)]
    q, k = (x.requires_grad_(True) for x in t[:2])
    freqs = rotary_frequencies(rot) if rot else torch.zeros(0, dtype=torch.float64)
    cu = torch.tensor([0, 5, 6, 6, 76, 109], dtype=torch.int64, device="cuda")
    outs = flash_rotary_varlen(q, k, freqs, cu, interleaved=interleaved, magnitude=1.25)
    pos = _event_positions(lens)[:, None]
    for got, x in zip(outs, (q, k)):
        _check(got, x, freqs, pos, interleaved, 1.25)
    for got, g in zip(torch.autograd.grad(outs, (q, k), t[2:]), t[2:]):
        _check(got, g, -freqs, pos, interleaved, 1.25)


@pytest.mark.parametrize("layout", ["bhld", "blhd"])
@pytest.mark.parametrize("where", ["rows", "given", "shared"])
@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP32, 48), (FP16, 10)])
def test_padded(dtype, dim, where, layout):
    b, n = 3, 37
    shape = (lambda h: (b, h, n, dim) if layout == "bhld" else (b, n, h, dim))
    q, k = (torch.randn(shape(h), device="cuda").to(dtype).requires_grad_(True) for h in (4, 2))
    freqs = rotary_frequencies(dim, scaling="linear", factor=4.0)
    pos = {"rows": None, "given": torch.randint(-50, 9999, (b, n)),
           "shared": torch.randint(0, 99, (n,))}[where]
    outs = flash_rotary(q, k, freqs, None if pos is None else pos.cuda(), layout=layout)
    ref = torch.arange(n).expand(b, n) if pos is None else pos.expand(b, n)
    ref = ref[:, None] if layout == "bhld" else ref[:, :, None]
    for got, x in zip(outs, (q, k)):
        _check(got, x, freqs, ref, False, 1.0)


@pytest.mark.parametrize("start", [65519, 999983, 2**31 - 41, 2**40])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_far_positions_keep_their_phase(dtype, start):
    # fp64 turns: off by 2^-52 of the angle, 2^-52 * 2^40 = 2^-12 turns at the
    # farthest, which is only held to that.
    x = torch.randn(40, 2, 64, device="cuda").to(dtype)
    freqs = rotary_frequencies(64, scaling="parts", factor=32.0)
    pos = start + torch.arange(40)
    got, none = flash_rotary_varlen(x, None, freqs, positions=pos.cuda(),
                                    magnitude=rotary_magnitude(32.0))
    assert none is None
    if start < 2**32:
        _check(got, x, freqs, pos[:, None], False, rotary_magnitude(32.0))
    else:
        ref = rotary_reference(x.double().cpu(), freqs, pos[:, None], False,
                               rotary_magnitude(32.0))
        assert (got.double().cpu() - ref).abs().max() <= 2.0**-8 * ref.abs().max() + 2.0**-7


def test_rows_of_no_event_are_copied():
    x = torch.randn(20, 2, 32, device="cuda")
    cu = torch.tensor([4, 9, 15], dtype=torch.int32, device="cuda")
    got, _ = flash_rotary_varlen(x, None, rotary_frequencies(32), cu, magnitude=2.0)
    assert torch.equal(got[:4], x[:4]) and torch.equal(got[15:], x[15:])
    _check(got[9:15], x[9:15], rotary_frequencies(32), torch.arange(6)[:, None], False, 2.0)


def test_strides_and_partial_gradients():
    fused = torch.randn(50, 8, 32, device="cuda", dtype=BF16)
    q, k, _ = fused.split((4, 2, 2), 1)
    freqs, cu = rotary_frequencies(32), torch.tensor([0, 20, 50], device="cuda")
    want = flash_rotary_varlen(q.contiguous(), k.contiguous(), freqs, cu)
    got = flash_rotary_varlen(q, k, freqs, cu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.zeros(50 * 4 * 32 + 1, device="cuda", dtype=BF16)[1:].view(50, 4, 32)
    odd.copy_(q)
    assert torch.equal(flash_rotary_varlen(odd, None, freqs, cu)[0], want[0])
    apart = torch.zeros(50, 4, 32, 2, device="cuda", dtype=BF16)[..., 0]
    apart.copy_(q)
    assert torch.equal(flash_rotary_varlen(apart, None, freqs, cu)[0], want[0])
    kl = k.contiguous().requires_grad_(True)
    outs = flash_rotary_varlen(q, kl, freqs, cu)
    (g,) = torch.autograd.grad(outs[1].float().sum(), kl)
    _check(g, torch.ones_like(kl), -freqs, _event_positions([20, 30])[:, None], False, 1.0)


def test_rotation_preserves_dot_products_of_equal_offsets():
    # <R_i q, R_j k> depends on i - j alone: shifting both positions changes
    # nothing but fp32 rounding (64 products of order 1 at 2^-21).
    q, k = (torch.randn(1, 1, 1, 64, device="cuda").expand(1, 1, 9, 64) for _ in range(2))
    freqs = rotary_frequencies(64)
    near = flash_rotary(q, k, freqs, torch.arange(9, device="cuda"))
    far = flash_rotary(q, k, freqs, torch.arange(9, device="cuda") + 123456)
    dots = [(a.double() @ b.double().transpose(-1, -2)) for a, b in (near, far)]
    scale = (q.abs().double() @ k.abs().double().transpose(-1, -2)).max()
    assert (dots[0] - dots[1]).abs().max() <= 2.0**-18 * scale


def test_graph_replay():
    x = torch.randn(64, 2, 32, device="cuda", dtype=BF16)
    freqs = rotary_frequencies(32).cuda()
    cu = torch.tensor([0, 30, 64], dtype=torch.int32, device="cuda")
    fixed = torch.zeros_like(x)
    flash_rotary_varlen(fixed, None, freqs, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = flash_rotary_varlen(fixed, None, freqs, cu)
    fixed.copy_(x)
    graph.replay()
    assert torch.equal(out, flash_rotary_varlen(x, None, freqs, cu)[0])


def test_offsets_past_32_bits():
    # 70 000 rows of 256 heads of 128: 2.3e9 elements.
    x = torch.zeros(70000, 256, 128, device="cuda", dtype=BF16)
    x[-3:] = torch.randn(3, 256, 128, device="cuda", dtype=BF16)
    freqs = rotary_frequencies(128)
    pos = torch.arange(70000, device="cuda")
    got, _ = flash_rotary_varlen(x, None, freqs, positions=pos)
    _check(got[-3:], x[-3:], freqs, pos[-3:, None], False, 1.0)
    assert got[:-3].count_nonzero() == 0


def test_outputs_may_be_the_inputs():
    # The C ABI allows it: every thread reads what it writes.
    import ctypes
    from flash_spacetime import _lib
    x = torch.randn(33, 5, 64, device="cuda", dtype=BF16)
    freqs = rotary_frequencies(48).cuda()
    pos = torch.arange(33, device="cuda")
    want, _ = flash_rotary_varlen(x, None, freqs, positions=pos)
    a = _lib.FstRotaryArgs()
    a.dtype, a.packed, a.heads, a.head_dim, a.pairs, a.positions_64 = _lib.FST_BF16, 1, 5, 64, 24, 1
    a.magnitude, a.total_rows, a.freqs, a.positions = 1.0, 33, freqs.data_ptr(), pos.data_ptr()
    a.q = a.q_out = _lib.FstRows(x.data_ptr(), 0, 64, 5 * 64)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.load().fst_rotary(ctypes.byref(a), stream), "fst_rotary")
    assert torch.equal(x, want)


def test_arguments_on_the_gpu_are_checked():
    q = torch.randn(2, 4, 9, 32, device="cuda")
    k = torch.randn(2, 2, 9, 32, device="cuda")
    freqs = rotary_frequencies(32)
    bad = [
        (dict(k=k.half()), "dtype"), (dict(k=k[:, :, :8]), "rows"), (dict(k=k[..., :16]), "rows"),
        (dict(k=k.cpu()), "CUDA"), (dict(freqs=rotary_frequencies(34)), "freqs"),
        (dict(freqs=freqs[None]), "freqs"), (dict(freqs=torch.arange(4)), "freqs"),
        (dict(freqs=freqs.clone().requires_grad_(True)), "grad"),
        (dict(positions=torch.zeros(9)), "integers"),
        (dict(positions=torch.zeros(2, 8, dtype=torch.int64)), "positions"),
        (dict(magnitude=float("inf")), "finite"), (dict(layout="packed"), "layout"),
    ]
    for change, text in bad:
        args = dict(q=q, k=k, freqs=freqs)
        args.update(change)
        with pytest.raises(ValueError, match=text):
            flash_rotary(**args)


def test_gradient_of_q_alone():
    q = torch.randn(30, 2, 32, device="cuda", requires_grad=True)
    freqs, cu = rotary_frequencies(32), torch.tensor([0, 12, 30], device="cuda")
    out, none = flash_rotary_varlen(q, None, freqs, cu, magnitude=0.5)
    g = torch.randn_like(q)
    (dq,) = torch.autograd.grad(out, q, g)
    assert none is None
    _check(dq, g, -freqs, _event_positions([12, 18])[:, None], False, 0.5)


def test_gradient_against_differences():
    # The op is linear: its difference along d is its value at d, up to the
    # fp32 rounding of 240 products of order 1.
    q, d, w = (torch.randn(10, 1, 24, device="cuda") for _ in range(3))
    q.requires_grad_(True)
    freqs, cu = rotary_frequencies(24), torch.tensor([0, 4, 10], device="cuda")
    (dq,) = torch.autograd.grad(flash_rotary_varlen(q, None, freqs, cu)[0], q, w)
    with torch.no_grad():
        far = (flash_rotary_varlen(q + d, None, freqs, cu)[0].double()
               - flash_rotary_varlen(q, None, freqs, cu)[0].double())
    want = (far * w.double()).sum()
    assert abs((dq.double() * d.double()).sum() - want) <= 2.0**-20 * 240 * 16


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype, dim, rot", [(BF16, 32, 32), (FP32, 64, 32), (FP16, 10, 6),
                                             (FP32, 7, 6), (BF16, 24, 16)])
def test_rows_of_no_event_keep_their_bits(dtype, dim, rot, interleaved):
    # Whatever such rows hold: infinities, NaN and zeros of either sign, whose
    # partner a rotation by 0 would change (x * 1 - y * 0).
    x = torch.randn(40, 3, dim, device="cuda").to(dtype)
    odd = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0, 0.0, 1.0], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    dead = torch.tensor([0, 1, 2, 30, 31, 39], device="cuda")
    pick = torch.randint(6, (6, 3, dim), device="cuda", generator=gen)
    x[dead] = odd[pick].to(dtype)
    cu = torch.tensor([3, 9, 30], dtype=torch.int32, device="cuda")
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    freqs = rotary_frequencies(rot)
    got, _ = flash_rotary_varlen(x, None, freqs, cu, interleaved=interleaved, magnitude=2.0)
    assert torch.equal(got[dead].view(bits), x[dead].view(bits))
    _check(got[3:30], x[3:30], freqs, _event_positions([6, 21])[:, None], interleaved, 2.0)
    leaf = torch.zeros_like(x).requires_grad_(True)
    out, _ = flash_rotary_varlen(leaf, None, freqs, cu, interleaved=interleaved)
    (grad,) = torch.autograd.grad(out, leaf, x)
    assert torch.equal(grad[dead].view(bits), x[dead].view(bits))


def _pi():
    """pi as a fraction, to 100 decimals: 16 atan(1/5) - 4 atan(1/239)."""
    unit = 10**110

    def atan(x):
        total, term, n = 0, unit // x, 1
        while term:
            total += term // n if n % 4 == 1 else -(term // n)
            term, n = term // (x * x), n + 2
        return total

    return Fraction(16 * atan(5) - 4 * atan(239), unit)


@pytest.mark.parametrize("start", [0, 10**6, 2**28, 2**31 - 20, 2**32, 2**40 + 3, 2**47 + 1])
def test_angles_against_exact_arithmetic(start):
    # Rows (1, 0) come back as (cos, sin) of position * freq, here in exact
    # rational arithmetic: within the 2^-22 of this file's header and the stated
    # 3 * 2^-53 of the angle.
    gen = torch.Generator().manual_seed(7)
    freqs = torch.cat((0.5 + torch.rand(24, generator=gen, dtype=torch.float64),
                       rotary_frequencies(16)))
    half = freqs.numel()
    pos = start + torch.arange(40)
    x = torch.zeros(40, 1, 2 * half, device="cuda")
    x[..., :half] = 1
    got, _ = flash_rotary_varlen(x, None, freqs, positions=pos.cuda())
    got = got[:, 0].double().cpu()
    two_pi = 2 * _pi()
    for i in range(40):
        for j in range(half):
            turns = int(pos[i]) * Fraction(freqs[j].item()) / two_pi
            angle = 2 * math.pi * float(turns - round(turns))
            bound = 2.0**-22 + 3 * 2.0**-53 * 2 * math.pi * float(turns)
            assert abs(got[i, j] - math.cos(angle)) <= bound
            assert abs(got[i, half + j] - math.sin(angle)) <= bound
