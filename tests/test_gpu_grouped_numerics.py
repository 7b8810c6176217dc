"""What rounding may not do to grouped-head attention: gradients that are
exactly zero, common offsets, and the range of 16-bit values."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime import (flash_grouped_attention, flash_grouped_attention_varlen,
                                 flash_rotary_varlen, grouped_attention_reference,
                                 rotary_frequencies, rotary_reference)

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# Tensor cores (one and two boxes of channels, a head that ends inside one), CUDA cores.
PATHS = [(BF16, 32), (BF16, 128), (FP16, 64), (FP16, 24), (BF16, 20), (FP16, 100), (FP32, 32),
         (FP32, 48), (FP32, 128)]


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _packed(lens, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, g = (torch.randn(sum(lens), h, dim, device="cuda", generator=gen).to(dtype)
                  for h in (heads, kv_heads, kv_heads, heads))
    return [t.requires_grad_(True) for t in (q, k, v)], g


# A row that sees one key has the weight 1 whatever its logit: its dq, and its
# share of dk, are 0, not the rounding of dP - D.


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", PATHS)
def test_events_of_one_row_have_no_gradient_of_q_and_k(dtype, dim, causal):
    leaves, g = _packed([1] * 150, 6, 2, dim, dtype)
    out = flash_grouped_attention_varlen(*leaves, _offsets([1] * 150), causal=causal)
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    assert dq.count_nonzero() == 0 and dk.count_nonzero() == 0
    assert torch.equal(out.detach(), leaves[2].detach().repeat_interleave(3, 1))
    want = g.double().unflatten(1, (2, 3)).sum(2)
    size = g.double().abs().unflatten(1, (2, 3)).sum(2)
    # One rounding, and P = 2^(x - lse2): x and lse2 are below 16 in size and
    # rounded three times, which leaves P off by less than 2^-18.
    assert ((dv.double() - want).abs()
            <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-18 * size).all()


@pytest.mark.parametrize("layout", ["bhld", "blhd"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", PATHS)
def test_padded_events_of_one_row(dtype, dim, causal, layout):
    shape = (lambda h: (5, h, 9, dim) if layout == "bhld" else (5, 9, h, dim))
    q, k, v = (torch.randn(shape(h), device="cuda").to(dtype).requires_grad_(True)
               for h in (4, 2, 2))
    out = flash_grouped_attention(q, k, v, [1, 0, 1, 1, 1], causal=causal, layout=layout)
    dq, dk, _ = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
    assert dq.count_nonzero() == 0 and dk.count_nonzero() == 0


@pytest.mark.parametrize("dtype, dim", PATHS)
def test_row_0_of_a_causal_event_has_no_gradient_of_q_and_k(dtype, dim):
    lens = [2, 1, 32, 33, 64, 130, 300]
    leaves, g = _packed(lens, 4, 2, dim, dtype, seed=1)
    cu = _offsets(lens)
    first = cu[:-1].long()
    out = flash_grouped_attention_varlen(*leaves, cu)
    dq = torch.autograd.grad(out, leaves[0], g)[0]
    assert dq[first].count_nonzero() == 0
    assert dq.count_nonzero() > 0.99 * (sum(lens) - len(lens)) * 4 * dim
    # A gradient at the first rows alone has nothing to change in q or k.
    only = torch.zeros_like(g)
    only[first] = g[first]
    out = flash_grouped_attention_varlen(*leaves, cu)
    dq, dk, dv = torch.autograd.grad(out, leaves, only)
    assert dq.count_nonzero() == 0 and dk.count_nonzero() == 0
    assert dv[first].count_nonzero() > 0


# Errors against float64 in units of what one rounding of the exact result
# leaves. Limits are those of a float64 model of the documented roundings (P,
# dS and the results), given with each, and a margin.


def _definition(q, k, v, g, causal, scale):
    """float64 out, dq, dk, dv of events ``[E, heads, n, D]``."""
    q, k, v, g = (t.detach().double() for t in (q, k, v, g))
    group = q.shape[1] // k.shape[1]
    q, g = (t.unflatten(1, (-1, group)) for t in (q, g))
    k, v = k[:, :, None], v[:, :, None]
    s = scale * (q @ k.transpose(-1, -2))
    if causal:
        s = s + torch.full(s.shape[-2:], float("-inf"), dtype=s.dtype, device=s.device).triu(1)
    p = s.softmax(-1)
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    return {"out": (p @ v).flatten(1, 2), "dq": scale * (ds @ k).flatten(1, 2),
            "dk": scale * (ds.transpose(-1, -2) @ q).sum(2),
            "dv": (p.transpose(-1, -2) @ g).sum(2)}


def _roundings(events, n, heads, kv_heads, dim, dtype, causal, v_mean=0.0, g_mean=0.0,
               g_scale=1.0, rows=slice(None), seed=0, k_mean=0.0):
    """Root mean square error of each result over that of rounding it once."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(h, mean=0.0, scale=1.0):
        t = torch.randn(events * n, h, dim, device="cuda", generator=gen)
        return (scale * (t + mean)).to(dtype)

    q, k, v = (t.requires_grad_(True) for t in (rand(heads), rand(kv_heads, k_mean),
                                                rand(kv_heads, v_mean)))
    g = rand(heads, g_mean, g_scale)
    out = flash_grouped_attention_varlen(q, k, v, _offsets([n] * events), causal=causal)
    got = dict(zip(("out", "dq", "dk", "dv"),
                   (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)))
    by_event = lambda t: t.unflatten(0, (events, n)).transpose(1, 2)  # noqa: E731
    want = _definition(*(by_event(t) for t in (q, k, v, g)), causal, dim**-0.5)
    ratios = {}
    for name, w in want.items():
        w, x = w[:, :, rows], by_event(got[name])[:, :, rows]
        ratios[name] = ((x.double() - w).norm() / (w.to(dtype).double() - w).norm()).item()
    return ratios


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP16, 64), (BF16, 128), (BF16, 32)])
@pytest.mark.parametrize("mean", [2.0, 8.0])
def test_a_common_offset_of_v_leaves_the_gradients_alone(dtype, dim, causal, mean):
    # D is that of the output whose weights sum to 1, so an offset of v cancels
    # in dP - D. Model: 1.1 for three keys (6 and 23 with weights that do not,
    # 4 and 15 with D from the rounded output); 1.45 for 256 (4 and 14).
    few = _roundings(300, 3, 4, 2, dim, dtype, causal, v_mean=mean, g_mean=1.0)
    assert few["dq"] <= 1.3 and few["dk"] <= 1.3 and few["out"] <= 1.1, few
    more = _roundings(8, 256, 4, 2, dim, dtype, causal, v_mean=mean, g_mean=1.0)
    assert more["dq"] <= 1.7 and more["dk"] <= 1.7 and more["out"] <= 1.1, more
    assert few["dv"] <= 1.5 and more["dv"] <= 1.5, (few, more)


@pytest.mark.parametrize("dtype, dim", [(BF16, 32), (FP16, 64), (BF16, 128)])
def test_output_of_long_rows_with_an_offset(dtype, dim):
    out = _roundings(1, 2500, 2, 1, dim, dtype, False, v_mean=8.0)["out"]
    assert out <= 1.1, out


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (BF16, 128), (FP16, 32), (FP16, 64)])
@pytest.mark.parametrize("n", [2, 3])
def test_gradients_of_two_and_three_keys_are_rounded_about_once(dtype, dim, causal, n):
    # Model: 1.1; 1.5 without the second part of dS; 1.9 with D from the
    # rounded output.
    got = _roundings(400, n, 4, 4, dim, dtype, causal, seed=n)
    assert got["dq"] <= 1.3 and got["dk"] <= 1.3, got


@pytest.mark.parametrize("g_scale", [1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("dim, causal", [(64, False), (64, True), (32, False), (128, True),
                                         (100, False)])
def test_fp16_gradients_of_long_events_keep_their_small_values(dim, causal, g_scale):
    # dS is about 1 / n of its row's gradient and falls below the normal range
    # of fp16 long before dq does. Model: 1.4; 2.8 (1e-2) and 8 (1e-3) with dS
    # in fp16 as it is.
    got = _roundings(1, 4096, 2, 1, dim, FP16, causal, g_scale=g_scale)
    assert got["dq"] <= 1.6 and got["dk"] <= 1.6 and got["dv"] <= 1.6, got


@pytest.mark.parametrize("dim", [64, 128])
def test_fp16_gradients_do_not_depend_on_other_events(dim):
    # Two events whose gradients are 2^12 apart, and an infinity in a third: each
    # has the bits that it has alone.
    lens, heads = [700, 1500, 40], 4
    leaves, g = _packed(lens, heads, 2, dim, FP16)
    g[700:2200] *= 2.0**-12
    g[2210] = float("inf")
    cu = _offsets(lens)
    out = flash_grouped_attention_varlen(*leaves, cu)
    all_events = torch.autograd.grad(out, leaves, g)
    for a, b in ((0, 700), (700, 2200)):
        own = [t.detach()[a:b].clone().requires_grad_(True) for t in leaves]
        out = flash_grouped_attention_varlen(*own, _offsets([b - a]))
        for x, y in zip(torch.autograd.grad(out, own, g[a:b]), all_events):
            assert torch.equal(x, y[a:b])
            assert x.isfinite().all() and x.count_nonzero() > 0


@pytest.mark.parametrize("dim", [64, 128])
def test_fp16_gradients_of_large_values_are_finite(dim):
    # |dS| reaches 1e6, far past fp16; dq and dk, with a small scale, do not.
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, g = (s * torch.randn(2, 2, 300, dim, device="cuda", generator=gen)
                  for s in (1, 1, 64, 512))
    leaves = [t.half().requires_grad_(True) for t in (q, k, v)]
    g = g.half()
    out = flash_grouped_attention(*leaves, scale=2.0**-9)
    got = torch.autograd.grad(out, leaves, g)
    want = _definition(*leaves, g, True, 2.0**-9)
    for name, x in zip(("dq", "dk", "dv"), got):
        w = want[name]
        assert x.isfinite().all() and w.abs().max() < 65504
        assert (x.double() - w).norm() <= 1.6 * (w.half().double() - w).norm()


@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (BF16, 128), (FP16, 32), (FP16, 128)])
@pytest.mark.parametrize("n", [32, 33, 64, 65, 200, 300])
def test_first_rows_of_causal_events_are_rounded_about_once(dtype, dim, n):
    # Rows that see few keys, whatever the event's length. Model: 1.1; 1.5
    # without the second part of dS.
    got = _roundings(100, n, 4, 2, dim, dtype, True, rows=slice(1, 4), seed=n)
    assert got["dq"] <= 1.3, got
    if n <= 33:
        got = _roundings(100, n, 4, 2, dim, dtype, True, seed=n)
        assert got["dq"] <= 1.3 and got["dk"] <= 1.3, got


# Sizes past those of the elementwise tests: long events, and enough of them
# that each block of the forward works through many.


@pytest.mark.parametrize("n, causal", [(5000, False), (9001, True)])
@pytest.mark.parametrize("dtype, dim, heads, kv_heads", [(BF16, 32, 2, 2), (FP16, 64, 2, 1),
                                                         (BF16, 128, 2, 1)])
def test_long_events(dtype, dim, heads, kv_heads, n, causal):
    # Model: out 1.4, dq and dk 1.45, dv 1.45 (over many keys P and dS are
    # rounded as often as the results).
    got = _roundings(1, n, heads, kv_heads, dim, dtype, causal)
    assert max(got.values()) <= 1.6, got


@pytest.mark.parametrize("dtype, dim", [(BF16, 32), (FP16, 64), (BF16, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_many_events(dtype, dim, causal):
    # 7200 items of the forward, some 25 to a block.
    got = _roundings(300, 130, 12, 4, dim, dtype, causal)
    assert max(got.values()) <= 1.6, got


@pytest.mark.parametrize("dtype, dim", [(BF16, 32), (FP16, 64), (BF16, 128), (FP32, 32)])
def test_an_event_has_the_same_bits_wherever_it_lies(dtype, dim):
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 400, (500,), generator=gen).tolist()
    leaves, g = _packed(lens, 6, 2, dim, dtype)
    starts = _offsets(lens)[:-1].tolist()
    order = torch.randperm(500, generator=gen).tolist()
    rows = torch.cat([torch.arange(starts[e], starts[e] + lens[e]) for e in order]).cuda()

    def run(leaves, g, lens):
        out = flash_grouped_attention_varlen(*leaves, _offsets(lens))
        return (out.detach(),) + torch.autograd.grad(out, leaves, g)

    moved = [t.detach()[rows].requires_grad_(True) for t in leaves]
    for a, b in zip(run(leaves, g, lens), run(moved, g[rows], [lens[e] for e in order])):
        assert torch.equal(a[rows], b)


@pytest.mark.parametrize("dtype, tol", [(BF16, 2e-2), (FP32, 1e-5)])
def test_rotary_then_attention_event_by_event(dtype, tol):
    # The two ops as they are used, each result of each event within the package's
    # parity tolerance of its own size; one row has no gradient of q and k.
    lens, heads, kv_heads, dim = [140, 1, 2, 263], 6, 2, 64
    (q, k, v), g = _packed(lens, heads, kv_heads, dim, dtype, seed=5)
    freqs, cu = rotary_frequencies(32), _offsets(lens)
    qr, kr = flash_rotary_varlen(q, k, freqs, cu)
    out = flash_grouped_attention_varlen(qr, kr, v, cu)
    got = (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)
    at = 0
    for n in lens:
        ref = [t.detach()[at:at + n].double().transpose(0, 1)[None].cpu().requires_grad_(True)
               for t in (q, k, v)]
        pos = torch.arange(n)[None, None]
        o = grouped_attention_reference(rotary_reference(ref[0], freqs, pos),
                                        rotary_reference(ref[1], freqs, pos), ref[2])
        grads = torch.autograd.grad(o, ref, g[at:at + n].double().transpose(0, 1)[None].cpu())
        for i, (a, b) in enumerate(zip(got, (o.detach(),) + grads)):
            a = a[at:at + n].transpose(0, 1).double().cpu()
            if n == 1 and i in (1, 2):
                assert a.count_nonzero() == 0
            else:
                assert (a - b[0]).norm() <= tol * b.norm()
        at += n


def test_fp16_powers_are_found_anew_on_every_replay():
    # The powers of two that keep dS within fp16 come from the values of the
    # replay, not of the capture.
    lens = [300, 41]
    leaves, g = _packed(lens, 4, 2, 64, FP16)
    cu = _offsets(lens)
    fixed = [torch.zeros_like(t) for t in (*leaves, g)]

    def run(q, k, v, g):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        return torch.autograd.grad(flash_grouped_attention_varlen(q, k, v, cu), (q, k, v), g)

    run(*fixed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*fixed)
    for g_scale, v_scale in ((1.0, 1.0), (2.0**-10, 1.0), (2.0**9, 2.0**3), (2.0**-3, 2.0**-8)):
        fresh = [leaves[0], leaves[1], leaves[2] * v_scale, g * g_scale]
        with torch.no_grad():
            for a, b in zip(fixed, fresh):
                a.copy_(b)
        graph.replay()
        for a, b in zip(run(*fresh), outs):
            assert torch.equal(a, b) and a.count_nonzero() > 0 and a.isfinite().all()


@pytest.mark.parametrize("dtype, dim", [(BF16, 32), (FP16, 128), (FP32, 32)])
def test_a_long_run_of_empty_events(dtype, dim):
    # The work list gives every event a position, an empty one too.
    leaves, g = _packed([200, 170], 2, 1, dim, dtype)
    cu = torch.cat((torch.zeros(60000), torch.full((60000,), 200.0),
                    torch.full((1000,), 370.0))).int().cuda()
    out = flash_grouped_attention_varlen(*leaves, cu)
    got = (out.detach(),) + torch.autograd.grad(out, leaves, g)
    out = flash_grouped_attention_varlen(*leaves, _offsets([200, 170]))
    want = (out.detach(),) + torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype, dim", [(FP16, 64), (FP16, 128), (BF16, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_gradient_row_that_is_not_finite_reaches_only_the_keys_it_sees(dtype, dim, value):
    # (dq and dk: dv may meet it in a tile, as 0 * NaN.)
    n, row = 500, 200
    leaves, g = _packed([n], 4, 2, dim, dtype)
    g *= 2.0**-6
    cu = _offsets([n])

    def run(x):
        g[row] = x
        out = flash_grouped_attention_varlen(*leaves, cu)
        return torch.autograd.grad(out, leaves[:2], g)

    for a, b, clean in zip(run(value), run(0.0), (slice(None), slice(row + 1, None))):
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[row] = False
        keep[:clean.start or 0] = False
        assert torch.equal(a[keep], b[keep]) and a[keep].count_nonzero() > 0
        assert not a[row].isfinite().all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype, dim", [(BF16, 64), (FP16, 64), (BF16, 128), (FP16, 72), (BF16, 24)])
@pytest.mark.parametrize("mean", [2.0, 8.0])
def test_a_common_offset_of_k_leaves_the_gradients_alone(dtype, dim, causal, mean):
    # dS sums to 0 over a row's keys but for its rounding, and what that leaves
    # times the offset is taken off dq again. Model: 1.1 for three keys (5.6 with
    # a mean of 8 left in), 1.5 for 256 (11).
    few = _roundings(300, 3, 4, 2, dim, dtype, causal, k_mean=mean)
    assert few["dq"] <= 1.3 and few["dk"] <= 1.3, few
    more = _roundings(8, 256, 4, 2, dim, dtype, causal, k_mean=mean)
    assert more["dq"] <= 1.7 and more["dk"] <= 1.7, more
