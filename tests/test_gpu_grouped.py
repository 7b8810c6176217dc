"""Grouped-head attention against its float64 definition, within bounds derived
from the documented roundings (grouped_cases)."""

import pytest
import torch

import grouped_cases as gc

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime import (flash_grouped_attention, flash_grouped_attention_varlen,
                                 flash_rotary_varlen, grouped_attention_reference,
                                 rotary_frequencies, rotary_reference)

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _offsets(lens, lead=0):
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _packed(lens, heads, kv_heads, dim, dtype, causal, lead=0, tail=0, **kw):
    events = gc.make_case(lens, heads, kv_heads, dim, dtype, causal, **kw)
    q, k, v, g = (gc.pack(events, x, lead, tail).cuda() for x in "qkvg")
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = flash_grouped_attention_varlen(q, k, v, _offsets(lens, lead), kw.get("scale"),
                                         causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), g)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads))
    total = lead + sum(lens)
    for name, t in got.items():
        assert torch.equal(t[:lead], torch.zeros_like(t[:lead])), name
        assert torch.equal(t[total:], torch.zeros_like(t[total:])), name
        at = lead
        for n, ev in zip(lens, events):
            if n:
                gc.check(t[at:at + n].transpose(0, 1), ev, name)
            at += n


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 48, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_packed_head_sizes(dtype, dim, causal):
    _packed([70, 1, 129, 300, 0, 64], 4, 2, dim, dtype, causal, seed=dim)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [1, 7, 20, 33, 64, 100, 128])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_packed_cuda_core_shapes(dtype, dim, causal):
    _packed([65, 1, 130, 0, 17], 3, 1, dim, dtype, causal, seed=dim)


@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255, 1, 256, 1, 257],
                                  [1] * 200, [513, 0, 0, 640], [0, 5, 0], [1100]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_packed_lengths(dim, causal, lens):
    _packed(lens, 2, 2, dim, BF16, causal, seed=len(lens))


@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP16, 32), (BF16, 128), (BF16, 24)])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_very_short_events(dtype, dim, causal):
    # Up to 32 rows dS is kept in two 16-bit parts (its rest is below 2^-16 of
    # it), so dq and dk are off by their own rounding, u |.|, and terms of the
    # order of fp32 (the bound's, with the rounding of P and dS taken out).
    lens = [2, 1, 3, 32, 7, 2, 31]
    events = gc.make_case(lens, 4, 2, dim, dtype, causal, seed=21)
    q, k, v, g = (gc.pack(events, x).cuda() for x in "qkvg")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = flash_grouped_attention_varlen(*leaves, _offsets(lens), causal=causal)
    dq, dk, _ = torch.autograd.grad(out, leaves, g)
    u, at = gc.HALF_STEP[dtype], 0
    for n, ev in zip(lens, events):
        for name, t, other in (("dq", dq, "k"), ("dk", dk, "q")):
            err = (t[at:at + n].transpose(0, 1).double().cpu() - ev[name]).abs()
            # dS <= |dP| + |D| <= 2 max |g| |v|; 2^-14 covers both parts' rest.
            size = 2 * ev["g"].double().norm(dim=-1).max() * ev["v"].double().norm(dim=-1).max()
            loose = 2.0**-14 * dim**-0.5 * size * ev[other].double().abs().max() * n * 2
            assert (err <= u * ev[name].abs() + loose).all(), (name, n)
        at += n


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (5, 1), (6, 3), (16, 2), (3, 3)])
@pytest.mark.parametrize("dim, dtype", [(32, BF16), (64, FP16), (128, BF16), (32, FP32)])
def test_head_groups(heads, kv_heads, dim, dtype):
    _packed([200, 31, 150], heads, kv_heads, dim, dtype, True, seed=heads)


@pytest.mark.parametrize("lead, tail", [(0, 1), (3, 0), (130, 257), (128, 128), (1000, 5)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_of_no_event_are_zero_and_never_read(dtype, lead, tail):
    # NaN around the events and (checked by the bounds) none of it inside.
    _packed([100, 140, 3], 2, 1, 64, dtype, True, lead=lead, tail=tail)


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 1e-3])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_scales(dtype, scale):
    _packed([150, 260], 2, 1, 32, dtype, True, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_large_logits(dtype):
    # Rows dominated by one key: logits spread over about +-60.
    _packed([150, 400], 2, 1, 64, dtype, True, spread=4.0)


def test_growing_logits_rescale():
    # Keys grow along the event, so the running maximum grows with every tile.
    events = gc.make_case([700], 2, 1, 64, BF16, True, seed=3)
    ev = events[0]
    ramp = torch.linspace(0.05, 6.0, 700, dtype=torch.float64)[None, :, None]
    ev["k"] = (ev["k"].double().abs() * ramp).to(BF16)
    ev["q"] = ev["q"].double().abs().to(BF16)
    res = gc.event_result(ev["q"].double(), ev["k"][0].double(), ev["v"][0].double(),
                          ev["g"].double(), 0.125, True, BF16)
    q, k, v, g = (gc.pack(events, x).cuda() for x in "qkvg")
    out = flash_grouped_attention_varlen(q, k, v, _offsets([700]))
    ev["out"], ev["bound"] = res["out"], res["bound"]
    gc.check(out.transpose(0, 1), ev, "out")


@pytest.mark.parametrize("layout", ["bhld", "blhd"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", [(BF16, 32), (FP16, 64), (BF16, 128), (FP32, 32),
                                        (BF16, 20)])
def test_padded(dtype, dim, causal, layout):
    lens, length = [150, 0, 1, 290, 128], 290
    events = gc.make_case(lens, 4, 2, dim, dtype, causal, seed=5)
    q, k, v, g = (gc.pad(events, x, length, layout).cuda() for x in "qkvg")
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = flash_grouped_attention(q, k, v, torch.tensor(lens, device="cuda"), causal=causal,
                                  layout=layout)
    grads = torch.autograd.grad(out, (q, k, v), g)
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads):
        t = t if layout == "bhld" else t.transpose(1, 2)
        for b, n in enumerate(lens):
            assert torch.equal(t[b, :, n:], torch.zeros_like(t[b, :, n:])), name
            if n:
                gc.check(t[b, :, :n], events[b], name)


def test_padded_length_forms_agree():
    lens = [20, 0, 33]
    q, k, v = (torch.randn(3, 2, 33, 32, device="cuda", dtype=BF16) for _ in range(3))
    mask = torch.arange(33)[None, :] >= torch.tensor(lens)[:, None]
    ref = flash_grouped_attention(q, k, v, torch.tensor(lens, device="cuda"))
    for form in (lens, torch.tensor(lens), torch.tensor(lens).short(), mask.cuda(),
                 torch.zeros(3, 33).masked_fill(mask, float("-inf")).cuda()):
        assert torch.equal(ref, flash_grouped_attention(q, k, v, form))
    assert torch.equal(ref, flash_grouped_attention(q, k, v, key_padding_mask=mask.cuda()))
    full = flash_grouped_attention(q, k, v, [33, 33, 33])
    assert torch.equal(full, flash_grouped_attention(q, k, v))
    assert torch.equal(full, flash_grouped_attention(q, k, v, [2**40, 99, 33]))


@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP32, 32), (BF16, 24)])
def test_strided_inputs_are_read_in_place(dtype, dim):
    heads, kv_heads, lens = 4, 2, [90, 200]
    events = gc.make_case(lens, heads, kv_heads, dim, dtype, True, seed=8)
    q, k, v, g = (gc.pack(events, x).cuda() for x in "qkvg")
    cu = _offsets(lens)
    fused = torch.cat((q, k, v), 1).requires_grad_(True)  # [T, H + 2 Hkv, D]
    parts = fused.split((heads, kv_heads, kv_heads), 1)
    out = flash_grouped_attention_varlen(*parts, cu)
    assert torch.equal(out, flash_grouped_attention_varlen(q, k, v, cu))
    (df,) = torch.autograd.grad(out, fused, g)
    qkv = [t.clone().requires_grad_(True) for t in (q, k, v)]
    ref = torch.autograd.grad(flash_grouped_attention_varlen(*qkv, cu), qkv, g)
    assert torch.equal(df, torch.cat(ref, 1))
    # Channels apart, rows off the 16-byte grid, an expanded gradient.
    wide = torch.zeros(q.shape[0], heads, dim, 2, dtype=dtype, device="cuda")
    wide[..., 0] = q
    assert torch.equal(out, flash_grouped_attention_varlen(wide[..., 0], k, v, cu))
    odd = torch.zeros(q.shape[0] * heads * dim + 1, dtype=dtype, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(out, flash_grouped_attention_varlen(odd, k, v, cu))
    got = torch.autograd.grad(flash_grouped_attention_varlen(*qkv, cu).sum(), qkv)
    want = torch.autograd.grad(flash_grouped_attention_varlen(*qkv, cu), qkv, torch.ones_like(q))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (BF16, 32), (FP32, 64)])
def test_deterministic_and_independent_of_the_batch(dtype, dim):
    # Bitwise equal run to run, and an event's rows do not depend on the others.
    lens = [333, 64, 700]
    t = [torch.randn(sum(lens), h, dim, device="cuda", dtype=dtype) for h in (6, 2, 2, 6)]

    def run(rows, lens):
        q, k, v, g = (x[rows].contiguous() for x in t)
        q, k, v = (x.requires_grad_(True) for x in (q, k, v))
        out = flash_grouped_attention_varlen(q, k, v, _offsets(lens))
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    one = run(slice(None), lens)
    for a, b in zip(one, run(slice(None), lens)):
        assert torch.equal(a, b)
    for a, b in zip(one, run(slice(333, 397), [64])):
        assert torch.equal(a[333:397], b)


def test_wrong_offsets_stay_inside_the_tensors():
    # Clamped, never followed outside; the results of such rows are unspecified.
    q, k, v = (torch.randn(300, 2, 32, device="cuda", dtype=BF16, requires_grad=True)
               for _ in range(3))
    for cu in ([-5, 100, 9000], [200, 100, 300], [0, 300, 20, 300], [0], [400, 500]):
        out = flash_grouped_attention_varlen(q, k, v, torch.tensor(cu, device="cuda"))
        torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    torch.cuda.synchronize()


def test_streams_and_graph_replay():
    lens = [100, 257, 40]
    cu = _offsets(lens)
    t = [torch.randn(sum(lens), h, 64, device="cuda", dtype=BF16) for h in (4, 2, 2, 4)]

    def run(q, k, v, g):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = flash_grouped_attention_varlen(q, k, v, cu)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    want = run(*t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    fixed = [torch.zeros_like(x) for x in t]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*fixed)
    for seed in (0, 1):
        fresh = [x if seed == 0 else x.flip(0) for x in t]
        for a, b in zip(fixed, fresh):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(run(*fresh), outs))


def test_empty_batches():
    for dtype in (BF16, FP32):
        q = torch.zeros(0, 4, 32, device="cuda", dtype=dtype, requires_grad=True)
        k = torch.zeros(0, 2, 32, device="cuda", dtype=dtype)
        out = flash_grouped_attention_varlen(q, k, k, _offsets([]))
        assert out.shape == (0, 4, 32)
        assert torch.autograd.grad(out.sum(), q)[0].shape == q.shape
        p = torch.zeros(0, 4, 16, 32, device="cuda", dtype=dtype)
        assert flash_grouped_attention(p, p, p).shape == p.shape
        p = torch.zeros(3, 4, 0, 32, device="cuda", dtype=dtype)
        assert flash_grouped_attention(p, p, p).shape == p.shape


def test_gradient_against_differences():
    # fp32 on the CUDA cores: (f(x + h d) - f(x - h d)) / 2h for a random
    # direction of all three inputs. Truncation is O(h^2) of third derivatives
    # of order 1, the differences round at 2^-24 |f| / h.
    gen = torch.Generator(device="cuda").manual_seed(4)
    t = [torch.randn(60, h, 32, device="cuda", generator=gen) for h in (2, 1, 1)]
    d = [torch.randn(x.shape, device="cuda", generator=gen) for x in t]
    w = torch.randn(60, 2, 32, device="cuda", generator=gen)
    cu = _offsets([25, 35])

    def f(sign, h=2.0**-7):
        args = [x + sign * h * y for x, y in zip(t, d)]
        return (flash_grouped_attention_varlen(*args, cu).double() * w).sum().item()

    leaves = [x.clone().requires_grad_(True) for x in t]
    grads = torch.autograd.grad(flash_grouped_attention_varlen(*leaves, cu), leaves, w)
    want = sum((a.double() * b).sum().item() for a, b in zip(grads, d))
    size = sum((a.double() * b).abs().sum().item() for a, b in zip(grads, d))
    got = (f(1) - f(-1)) * 2.0**6
    assert abs(got - want) <= 1e-3 * size


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rotary_then_attention(dtype):
    # The two ops as they are used: q and k rotated, then causal attention,
    # against float64 autograd through both definitions.
    lens, heads, kv_heads, dim = [140, 1, 263], 6, 2, 64
    total = sum(lens)
    freqs = rotary_frequencies(32)
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(total, h, dim, generator=gen, dtype=torch.float64).to(dtype)
                  for h in (heads, kv_heads, kv_heads, heads))
    dev = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    cu = _offsets(lens)
    qr, kr = flash_rotary_varlen(dev[0], dev[1], freqs, cu)
    out = flash_grouped_attention_varlen(qr, kr, dev[2], cu)
    got = (out.detach(),) + torch.autograd.grad(out, dev, g.cuda())
    at, tol = 0, {BF16: 2e-2, FP32: 1e-5}[dtype]
    for n in lens:
        ref = [t[at:at + n].double().transpose(0, 1)[None].requires_grad_(True) for t in (q, k, v)]
        pos = torch.arange(n)[None, None]
        o = grouped_attention_reference(rotary_reference(ref[0], freqs, pos),
                                        rotary_reference(ref[1], freqs, pos), ref[2])
        grads = torch.autograd.grad(o, ref, g[at:at + n].double().transpose(0, 1)[None])
        for a, b in zip(got, (o.detach(),) + grads):
            a = a[at:at + n].transpose(0, 1).double().cpu()
            # Normwise, the tolerance of the package's parity tests; an event
            # of one row has dq = dk = 0 up to the rounding of D.
            assert (a - b[0]).norm() <= tol * (b.norm() + g[at:at + n].double().norm())
        at += n


def test_offsets_past_32_bits():
    # 70 000 rows of 256 heads of 128: 2.3e9 elements. Two short events, one at
    # either end; every other row is of no event.
    total, heads, dim = 70000, 256, 128
    q = torch.zeros(total, heads, dim, device="cuda", dtype=BF16)
    k, v = (torch.randn(total, 1, dim, device="cuda", dtype=BF16) for _ in range(2))
    rows = torch.cat((torch.arange(40), torch.arange(total - 150, total))).cuda()
    q[rows] = torch.randn(190, heads, dim, device="cuda", dtype=BF16)
    g = torch.ones_like(q)
    cu = torch.tensor([0, 40, 40, 40], dtype=torch.int32, device="cuda")
    late = torch.tensor([total - 150, total], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for offsets, part, lens in ((cu, slice(0, 40), [40]), (late, slice(total - 150, total), [150])):
        out = flash_grouped_attention_varlen(q, k, v, offsets)
        got = (out.detach(),) + torch.autograd.grad(out, leaves, g)
        small = [t[part].detach().clone().requires_grad_(True) for t in (q, k, v)]
        ref = flash_grouped_attention_varlen(*small, _offsets(lens))
        want = (ref.detach(),) + torch.autograd.grad(ref, small, g[part])
        for a, b in zip(got, want):
            assert torch.equal(a[part], b)
            assert a.flatten().count_nonzero() == b.count_nonzero()


def test_two_streams_at_once():
    # Calls that overlap share nothing: each gives what it gives alone.
    lens = [700, 129, 40]
    cu = _offsets(lens)
    sets = [[torch.randn(sum(lens), h, d, device="cuda", dtype=t) for h in (4, 2, 2, 4)]
            for d, t in ((64, BF16), (128, FP16))]

    def run(q, k, v, g):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = flash_grouped_attention_varlen(q, k, v, cu)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, t) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(run(*t))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP16, 128), (FP32, 32)])
def test_a_nan_row_stays_visible(dtype, dim):
    # A NaN in row 5 of k reaches every row of its event that sees it, and no
    # row of another event.
    q, k, v = (torch.randn(300, 2, dim, device="cuda", dtype=dtype) for _ in range(3))
    cu = _offsets([100, 200])
    clean = flash_grouped_attention_varlen(q, k, v, cu, causal=False)
    k[5] = float("nan")
    out = flash_grouped_attention_varlen(q, k, v, cu, causal=False)
    assert out[:100].isnan().all()
    assert torch.equal(out[100:], clean[100:])


def test_gradients_are_differentiable_once():
    q, k, v = (torch.randn(20, 1, 32, device="cuda", requires_grad=True) for _ in range(3))
    out = flash_grouped_attention_varlen(q, k, v, _offsets([20]))
    (dq,) = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)


def test_arguments_on_the_gpu_are_checked():
    q = torch.randn(2, 4, 9, 32, device="cuda", dtype=BF16)
    k = torch.randn(2, 2, 9, 32, device="cuda", dtype=BF16)
    bad = [
        (dict(k=k.float()), "dtype"), (dict(k=k[:, :, :8], v=k[:, :, :8]), "rows"),
        (dict(v=k[..., :16]), "rows"), (dict(k=k.cpu()), "CUDA"),
        (dict(k=torch.cat((k, k[:, :1]), 1), v=torch.cat((k, k[:, :1]), 1)), "multiple"),
        (dict(layout="packed"), "varlen"), (dict(layout="x"), "layout"),
        (dict(seqlens=torch.tensor([1.0, 2.0])), "integers"), (dict(seqlens=[1, 2, 3]), "seqlens"),
        (dict(seqlens=torch.zeros(2, 8, dtype=torch.bool)), "mask"),
        (dict(seqlens=[1, 2], key_padding_mask=torch.zeros(2, 9, dtype=torch.bool)), "not both"),
        (dict(q=torch.randn(2, 4, 9, 136, device="cuda"),
              k=torch.randn(2, 4, 9, 136, device="cuda"),
              v=torch.randn(2, 4, 9, 136, device="cuda")), "128"),
        (dict(scale=float("nan")), "finite"),
    ]
    for change, text in bad:
        args = dict(q=q, k=k, v=k)
        args.update(change)
        with pytest.raises(ValueError, match=text):
            flash_grouped_attention(**args)
    packed = [t.transpose(1, 2).flatten(0, 1) for t in (q, k, k)]
    for cu in (torch.tensor([[0, 9]]), torch.tensor([0.0, 9.0]), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError):
            flash_grouped_attention_varlen(*packed, cu)
