"""Cases of the grouped-head attention and rotary position operators.

``listed()`` and ``draw()`` describe cases as plain dicts; ``prepare`` makes
a case's inputs on the GPU; ``run`` makes one pass, either in plain torch
operations (``own`` false) or through ``flash_spacetime`` (``own`` true);
``exact`` gives the same outputs from the definitions in float64; ``work``
counts the bytes and operations a pass cannot do without.

Two operators:

* ``attention``: softmax attention over events (sequences) of different
  lengths, packed ``[T, H, Dh]`` or padded ``[B, H, L, Dh]`` /
  ``[B, L, H, Dh]``; the queries of ``H / Hkv`` heads share one key and value
  head; causal or not; forward only, or forward with dq, dk, dv.
* ``rotary``: rotation of the first ``R`` of the ``Dh`` channels of q and k
  by ``position * freqs``, channels paired by halves or interleaved,
  frequencies scaled for long contexts; forward only, or with its gradient.
"""

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # A handful of short events, as an online filter sees them: latency.
        dict(name="attn_few_events", op="attention", layout="packed", dtype="bf16", heads=12,
             kv_heads=12, dim=32, causal=False, train=False, events=4, longest=48,
             spread="uniform", lens_seed=11),
        # The default benchmark's batch (256 events, lognormal lengths with
        # median 120, at most 768; 12 heads of 32) through a block without the
        # pair term, trained.
        dict(name="attn_events_train", op="attention", layout="packed", dtype="bf16", heads=12,
             kv_heads=12, dim=32, causal=False, train=True, events=256, longest=768,
             spread="lognormal", lens_seed=1),
        # Ragged prompts, causal, four query heads to a key head: inference.
        dict(name="attn_prompts", op="attention", layout="packed", dtype="bf16", heads=32,
             kv_heads=8, dim=128, causal=True, train=False, events=7, longest=4096,
             spread="uniform", lens_seed=5),
        # A training batch of packed documents at the wide head size.
        dict(name="attn_documents_train", op="attention", layout="packed", dtype="bf16", heads=16,
             kv_heads=4, dim=128, causal=True, train=True, events=5, longest=4096,
             spread="uniform", lens_seed=6),
        # One event of the longest length the framework is run at, in fp16.
        dict(name="attn_long_train", op="attention", layout="packed", dtype="fp16", heads=8,
             kv_heads=8, dim=64, causal=True, train=True, events=1, longest=16384,
             spread="full", lens_seed=0),
        # The sweep shape (L = 1024, 8 heads of 64), padded row-major, two
        # query heads to a key head, some events short.
        dict(name="attn_padded_train", op="attention", layout="blhd", dtype="bf16", heads=8,
             kv_heads=4, dim=64, causal=True, train=True, events=24, longest=1024,
             spread="uniform", lens_seed=3),
        # The fp32 parity configuration: 4 events padded to 128, 12 heads of 32.
        dict(name="attn_fp32_train", op="attention", layout="bhld", dtype="fp32", heads=12,
             kv_heads=12, dim=32, causal=True, train=True, events=4, longest=128,
             spread="uniform", lens_seed=4),
        # Few short events before attention: latency.
        dict(name="rotary_few_events", op="rotary", layout="packed", dtype="bf16", heads=12,
             kv_heads=12, dim=32, rot=32, interleaved=False, scaling="none", factor=1.0, far=0,
             train=False, events=4, longest=48, spread="uniform", lens_seed=11),
        # The default benchmark's batch, half of each head rotated, pairs
        # interleaved, with the gradient.
        dict(name="rotary_events_train", op="rotary", layout="packed", dtype="bf16", heads=12,
             kv_heads=12, dim=32, rot=16, interleaved=True, scaling="none", factor=1.0, far=0,
             train=True, events=256, longest=768, spread="lognormal", lens_seed=1),
        # Long prompts far into a context of a million tokens, frequencies
        # scaled by parts, 32 query and 8 key heads of 128.
        dict(name="rotary_far_prompts", op="rotary", layout="packed", dtype="bf16", heads=32,
             kv_heads=8, dim=128, rot=128, interleaved=False, scaling="parts", factor=32.0,
             far=1000003, train=False, events=3, longest=16384, spread="uniform", lens_seed=2),
        # A padded fp32 batch, head size 48, linear scaling, with the gradient.
        dict(name="rotary_padded_fp32_train", op="rotary", layout="bhld", dtype="fp32", heads=12,
             kv_heads=4, dim=48, rot=48, interleaved=False, scaling="linear", factor=4.0, far=0,
             train=True, events=33, longest=511, spread="uniform", lens_seed=8),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A case of the ranges the listed ones stand for."""
    op = rng.choice(["attention", "attention", "rotary"])
    case = dict(op=op)
    case["layout"] = rng.choice(["packed", "packed", "bhld", "blhd"])
    case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 8, 12])
    case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 4, 5])
    case["train"] = rng.random() < 0.6
    case["spread"] = rng.choice(["uniform", "lognormal", "full"])
    case["lens_seed"] = rng.randrange(1 << 20)
    if op == "attention":
        case["dim"] = rng.choice([16, 24, 32, 40, 48, 64, 64, 80, 96, 128, 128])
        case["causal"] = rng.random() < 0.6
        case["longest"] = _log_int(rng, 1, 8192 if case["dtype"] != "fp32" else 1500)
        limit = 4.0e11 if case["dtype"] != "fp32" else 2.0e10
    else:
        case["dim"] = rng.choice([16, 32, 48, 64, 80, 96, 128])
        case["rot"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2, case["dim"] // 4])
        case["interleaved"] = rng.random() < 0.4
        case["scaling"] = rng.choice(["none", "linear", "base", "parts"])
        case["factor"] = 1.0 if case["scaling"] == "none" else rng.choice([2.0, 8.0, 32.0])
        case["far"] = rng.choice([0, 0, 65521, 1000003])
        case["longest"] = _log_int(rng, 1, 16384)
        limit = 1.6e8
    case["events"] = _log_int(rng, 1, 64)
    # No more work, and no more memory, than the largest listed cases.
    def too_large():
        values = _rows(case) * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return work(case)["flops"] > limit or values > 1.5e8

    while case["events"] > 1 and too_large():
        case["events"] = (case["events"] + 1) // 2
    while too_large():
        case["longest"] = max(1, case["longest"] * 3 // 4)
    return case


def _lengths(case):
    n, longest = case["events"], case["longest"]
    if case["spread"] == "full":
        return [longest] * n
    rng = random.Random(case["lens_seed"])
    if case["spread"] == "uniform":
        lens = [rng.randint(1, longest) for _ in range(n)]
        lens[rng.randrange(n)] = longest
        return lens
    median = max(1.0, 120.0 * longest / 768.0)
    return [min(longest, max(1, round(median * math.exp(1.2 * rng.gauss(0.0, 1.0)))))
            for _ in range(n)]


def _rows(case):
    if case["layout"] == "packed":
        return sum(_lengths(case))
    return case["events"] * case["longest"]


def _shape(case, heads):
    b, n, d = case["events"], case["longest"], case["dim"]
    if case["layout"] == "packed":
        return (_rows(case), heads, d)
    return (b, heads, n, d) if case["layout"] == "bhld" else (b, n, heads, d)


def _frequencies(case):
    """float64 ``[R/2]`` angle per position of each channel pair."""
    half = case["rot"] // 2
    base, factor = 10000.0, case["factor"]
    if case["scaling"] == "base" and case["rot"] > 2:
        base *= factor ** (case["rot"] / (case["rot"] - 2))
    freqs = base ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        freqs = freqs / factor
    if case["scaling"] == "parts":
        # Pairs that turn more than 32 times over the trained 4096 positions
        # keep their frequency, those below one turn are divided by the
        # factor, a linear ramp between.
        turns = 4096 * freqs / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
    return freqs


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def rand(heads):
        return torch.randn(_shape(case, heads), generator=gen, device="cuda").to(dtype)

    state = {"case": case}
    names = [("q", "heads"), ("k", "kv_heads")]
    grads = [("gq", "heads"), ("gk", "kv_heads")]
    if case["op"] == "attention":
        names.append(("v", "kv_heads"))
        grads = [("g", "heads")]
    for name, heads in names:
        state[name] = rand(case[heads])
    if case["train"]:
        for name, _ in names:
            state[name].requires_grad_(True)
        for name, heads in grads:
            state[name] = rand(case[heads])
    lens = _lengths(case)
    if case["layout"] == "packed":
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        state["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        state["bounds"] = list(zip(cu[:-1], cu[1:]))
    elif case["op"] == "attention":
        state["lens"] = lens
        state["seqlens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["op"] == "rotary":
        state["freqs"] = _frequencies(case).cuda()
        state["positions"] = None
        if case["far"]:
            # Documents that begin anywhere in a long context.
            rng = random.Random(seed)
            if case["layout"] == "packed":
                parts = [torch.arange(n) + rng.randrange(case["far"]) for n in lens]
                state["positions"] = torch.cat(parts).to("cuda", torch.int32)
            else:
                parts = [torch.arange(case["longest"]) + rng.randrange(case["far"]) for _ in lens]
                state["positions"] = torch.stack(parts).to("cuda", torch.int32)
    return state


# ---- the calls a user makes -------------------------------------------------


def _run_own(state):
    import sys
    if "flash-spacetime_b200" not in sys.path:
        sys.path.insert(0, "flash-spacetime_b200")
    import flash_spacetime as fst
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "attention":
            q, k, v = state["q"], state["k"], state["v"]
            if case["layout"] == "packed":
                out = fst.flash_grouped_attention_varlen(q, k, v, state["cu"],
                                                         causal=case["causal"])
            else:
                out = fst.flash_grouped_attention(q, k, v, state["seqlens"],
                                                  causal=case["causal"], layout=case["layout"])
            if not case["train"]:
                return out
            return (out.detach(),) + torch.autograd.grad(out, (q, k, v), state["g"])
        q, k = state["q"], state["k"]
        if case["layout"] == "packed":
            outs = fst.flash_rotary_varlen(q, k, state["freqs"], state["cu"], state["positions"],
                                           interleaved=case["interleaved"],
                                           magnitude=_magnitude(case))
        else:
            outs = fst.flash_rotary(q, k, state["freqs"], state["positions"],
                                    layout=case["layout"], interleaved=case["interleaved"],
                                    magnitude=_magnitude(case))
        if not case["train"]:
            return outs
        grads = torch.autograd.grad(outs, (q, k), (state["gq"], state["gk"]))
        return tuple(o.detach() for o in outs) + grads


# ---- the plain form ---------------------------------------------------------


def _events(state, t):
    """Each event's rows of ``t`` as a ``[heads, length, Dh]`` view."""
    case = state["case"]
    if case["layout"] == "packed":
        return [t[a:b].transpose(0, 1) for a, b in state["bounds"]]
    if case["layout"] == "bhld":
        return [t[i, :, :n] for i, n in enumerate(state["lens"])]
    return [t[i, :n].transpose(0, 1) for i, n in enumerate(state["lens"])]


def _plain_event(q, k, v, g, causal, scale):
    """Attention of one event: q ``[h, G, n, D]`` on k and v ``[h, 1, n, D]``."""
    n = q.shape[2]
    s = (q * scale) @ k.transpose(2, 3)
    if causal:
        pos = torch.arange(n, device=q.device)
        s = s.masked_fill(pos[None, :] > pos[:, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = p @ v
    if g is None:
        return (out,)
    dv = (p.transpose(2, 3) @ g).sum(1)
    dp = g @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(2, 3) @ (q * scale)).sum(1)
    return out, dq, dk, dv


def _plain_attention(state):
    case = state["case"]
    q, k, v = (state[x].detach() for x in "qkv")
    train = case["train"]
    outs = [torch.zeros_like(t) for t in ((q, q, k, v) if train else (q,))]
    group = case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    gs = _events(state, state["g"]) if train else [None] * case["events"]
    views = [_events(state, o) for o in outs]
    for e, rows in enumerate(zip(_events(state, q), _events(state, k), _events(state, v), gs)):
        # As many key heads at once as keep the logits within 1 GB.
        step = max(1, (1 << 28) // (group * rows[0].shape[1] ** 2))
        for h in range(0, case["kv_heads"], step):
            kv = slice(h, min(h + step, case["kv_heads"]))
            mine = slice(kv.start * group, kv.stop * group)
            qe, ge = (None if t is None else t[mine].float().unflatten(0, (-1, group))
                      for t in (rows[0], rows[3]))
            ke, ve = (t[kv].float().unsqueeze(1) for t in rows[1:3])
            got = _plain_event(qe, ke, ve, ge, case["causal"], scale)
            for i, part in enumerate(got):
                if i < 2:
                    views[i][e][mine] = part.flatten(0, 1).to(q.dtype)
                else:
                    views[i][e][kv] = part.to(q.dtype)
    return tuple(outs) if train else outs[0]


def _positions(state):
    """Position of each row, shaped to broadcast over heads and pairs."""
    case = state["case"]
    pos = state["positions"]
    if case["layout"] == "packed":
        if pos is None:
            pos = torch.cat([torch.arange(b - a, device="cuda") for a, b in state["bounds"]])
        return pos[:, None, None]
    if pos is None:
        pos = torch.arange(case["longest"], device="cuda").expand(case["events"], -1)
    return pos[:, None, :, None] if case["layout"] == "bhld" else pos[:, :, None, None]


def _plain_rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    y = x.float()
    a, b = ((y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved
            else (y[..., :rot // 2], y[..., rot // 2:rot]))
    out = y.clone()
    lo, hi = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = lo, hi
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = lo, hi
    return out.to(x.dtype)


def _plain_rotary(state):
    case = state["case"]
    angle = _positions(state).double() * state["freqs"]
    mag = _magnitude(case)
    cos, sin = (torch.cos(angle) * mag).float(), (torch.sin(angle) * mag).float()
    flip = case["interleaved"]
    outs = [_plain_rotate(state[x].detach(), cos, sin, flip) for x in ("q", "k")]
    if case["train"]:
        outs += [_plain_rotate(state[x], cos, -sin, flip) for x in ("gq", "gk")]
    return tuple(outs)


def run(state):
    if own:
        return _run_own(state)
    if state["case"]["op"] == "attention":
        return _plain_attention(state)
    return _plain_rotary(state)


# ---- the definitions in float64 ---------------------------------------------


def _exact_attention(case, state):
    q, k, v = (state[x].detach().double().requires_grad_(case["train"]) for x in "qkv")
    group = case["heads"] // case["kv_heads"]
    gout = state["g"].double() if case["train"] else None
    full = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v)]

    def rows(t, e, h):
        if case["layout"] == "packed":
            a, b = state["bounds"][e]
            return t[a:b, h]
        n = state["lens"][e]
        return t[e, h, :n] if case["layout"] == "bhld" else t[e, :n, h]

    for e in range(case["events"]):
        for h in range(case["heads"]):
            qs, ks, vs = (rows(t, e, i).detach().requires_grad_(case["train"])
                          for t, i in ((q, h), (k, h // group), (v, h // group)))
            logits = torch.einsum("id,jd->ij", qs, ks) / math.sqrt(case["dim"])
            if case["causal"]:
                logits = logits + torch.full_like(logits.detach(), float("-inf")).triu_(1)
            out = torch.softmax(logits, 1) @ vs
            rows(full, e, h).copy_(out.detach())
            if case["train"]:
                parts = torch.autograd.grad(out, (qs, ks, vs), rows(gout, e, h))
                for t, i, part in zip(grads, (h, h // group, h // group), parts):
                    rows(t, e, i).add_(part)
    return (full, *grads) if case["train"] else full


def _exact_rotary(case, state):
    pos = _positions(state).double()
    turn = torch.polar(torch.full_like(pos * state["freqs"], _magnitude(case)),
                       pos * state["freqs"])

    def rotate(x, turn):
        x = x.detach().double()
        head, tail = x[..., :case["rot"]], x[..., case["rot"]:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(*head.chunk(2, -1)) * turn
            head = torch.cat((z.real, z.imag), -1)
        return torch.cat((head, tail), -1)

    outs = [rotate(state["q"], turn), rotate(state["k"], turn)]
    if case["train"]:
        outs += [rotate(state["gq"], turn.conj()), rotate(state["gk"], turn.conj())]
    return tuple(outs)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    if case["events"] * case["heads"] > 12000:  # over about 20 seconds of launches
        return None
    return _exact_attention(case, state)


def work(case):
    rows, d = _rows(case), case["dim"]
    size = 4 if case["dtype"] == "fp32" else 2
    lens = _lengths(case)
    if case["op"] == "attention":
        # Only the events' own rows have to be read; padding rows are written 0.
        live = sum(lens)
        qn, kn = live * case["heads"] * d * size, live * case["kv_heads"] * d * size
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens) * case["heads"]
        out = rows * case["heads"] * d * size
        if not case["train"]:
            return {"bytes": qn + 2 * kn + out, "flops": 4 * d * pairs}
        grads = rows * (case["heads"] + 2 * case["kv_heads"]) * d * size
        return {"bytes": 2 * qn + 2 * kn + out + grads, "flops": 14 * d * pairs}
    values = rows * (case["heads"] + case["kv_heads"])
    passes = 2 if case["train"] else 1
    moved = 2 * values * d * size * passes + (rows * 4 if case["far"] else 0)
    return {"bytes": moved, "flops": 3 * values * case["rot"] * passes}
