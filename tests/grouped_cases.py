"""Inputs, float64 results and elementwise error bounds of the grouped-head
attention tests.

The bounds are first-order and worst-case, from the roundings that the kernels
document. With u half a step of the tensors' type and g the fp32 summation
constant below, written for one head, |.| and products elementwise:

* P is rounded to the type before P v (16-bit types):
    d_out = (u + g) P |v| + u |out|
* D_i = dO_i . out_i uses the stored (rounded) out:
    d_D = |dO| . d_out + g |dO| . |out|
* dS = P (dP - D) is rounded to the type before it multiplies k or q:
    d_dS = P (d_D + g |dO| |v|^T) + (u + 2 g) |dS| + g P (|dP| + |D|)
* d_dv = (u + g) P^T |dO| + u |dv|
* d_dq = scale (d_dS |k| + g |dS| |k|) + u |dq|, d_dk likewise with |q|.

g covers every fp32 step of a result: sums of at most n terms (n 2^-24 each,
over the keys, the queries of a group or the channels), the logit's own
rounding in the exponent (2^-24 times |s| and its sum of Dh terms), and the
few ulp of exp2 and of the division.
"""

from typing import Dict, List, Optional, Sequence

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def event_result(q, k, v, g, scale: float, causal: bool, dtype: torch.dtype) -> Dict:
    """float64 out, dq, dk, dv of one event and head group, with their bounds.

    q, g: ``[G, n, D]``; k, v: ``[n, D]`` (float64 values of ``dtype`` tensors).
    """
    n, dim = k.shape
    s = scale * (q @ k.T)
    seen = torch.ones(n, n, dtype=torch.bool)
    if causal:
        seen = seen.tril()
    s = s.masked_fill(~seen, float("-inf"))
    p = s.softmax(-1)
    out = p @ v
    dp = g @ v.T
    d = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - d)
    res = {"out": out, "dv": (p.transpose(1, 2) @ g).sum(0), "dq": scale * (ds @ k),
           "dk": scale * (ds.transpose(1, 2) @ q).sum(0)}
    u = HALF_STEP[dtype]
    reach = (abs(scale) * (q.abs() @ k.abs().T)).masked_fill(~seen, 0).max().item()
    gam = 2.0**-24 * (n * q.shape[0] + 2 * dim + 64 + (dim + 4) * reach)
    up = u if dtype != torch.float32 else 0.0
    pv = p @ v.abs()
    e_out = (up + gam) * pv + u * out.abs()
    e_d = (g.abs() * e_out).sum(-1, keepdim=True) + gam * (g.abs() * out.abs()).sum(-1, keepdim=True)
    e_ds = (p * (e_d + gam * (g.abs() @ v.abs().T)) + (up + 2 * gam) * ds.abs()
            + gam * p * (dp.abs() + d.abs()))
    e_ds = e_ds + gam * ds.abs()
    tiny = torch.finfo(dtype).tiny * n
    res["bound"] = {
        "out": e_out + tiny,
        "dv": ((up + gam) * (p.transpose(1, 2) @ g.abs())).sum(0) + u * res["dv"].abs() + tiny,
        "dq": abs(scale) * (e_ds @ k.abs()) + u * res["dq"].abs() + tiny,
        "dk": abs(scale) * (e_ds.transpose(1, 2) @ q.abs()).sum(0) + u * res["dk"].abs() + tiny,
    }
    return res


def make_case(lens: Sequence[int], heads: int, kv_heads: int, dim: int, dtype: torch.dtype,
              causal: bool, seed: int = 0, scale: Optional[float] = None, spread: float = 1.0):
    """Per-event inputs (rounded to ``dtype``) and their float64 results."""
    gen = torch.Generator().manual_seed(seed)
    events: List[Dict] = []
    group = heads // kv_heads
    used = dim**-0.5 if scale is None else scale

    def rand(h, n):
        x = spread * torch.randn(h, n, dim, generator=gen, dtype=torch.float64)
        return x.to(dtype)

    for n in lens:
        ev = {"q": rand(heads, n), "k": rand(kv_heads, n), "v": rand(kv_heads, n),
              "g": rand(heads, n)}
        names = ("out", "dq", "dk", "dv")
        res = {name: [] for name in names}
        bound = {name: [] for name in names}
        for h in range(kv_heads if n else 0):
            mine = slice(h * group, (h + 1) * group)
            r = event_result(ev["q"][mine].double(), ev["k"][h].double(), ev["v"][h].double(),
                             ev["g"][mine].double(), used, causal, dtype)
            for name in names:
                res[name].append(r[name] if r[name].dim() == 3 else r[name][None])
                bound[name].append(r["bound"][name] if r[name].dim() == 3
                                   else r["bound"][name][None])
        if n:
            ev.update({name: torch.cat(res[name]) for name in names})
            ev["bound"] = {name: torch.cat(bound[name]) for name in names}
        events.append(ev)
    return events


def pack(events, name: str, lead: int = 0, tail: int = 0, fill: float = float("nan")):
    """``[T, heads, D]`` of the events, with rows of ``fill`` around them."""
    parts = [ev[name].transpose(0, 1) for ev in events]
    like = parts[0]
    pad = lambda n: torch.full((n,) + like.shape[1:], fill, dtype=like.dtype)  # noqa: E731
    return torch.cat([pad(lead)] + parts + [pad(tail)])


def pad(events, name: str, length: int, layout: str, fill: float = float("nan")):
    """Padded ``[B, heads, L, D]`` or ``[B, L, heads, D]``, padding rows ``fill``."""
    first = events[0][name]
    out = torch.full((len(events), first.shape[0], length, first.shape[2]), fill,
                     dtype=first.dtype)
    for b, ev in enumerate(events):
        out[b, :, :ev[name].shape[1]] = ev[name]
    return out if layout == "bhld" else out.transpose(1, 2).contiguous()


def check(got: torch.Tensor, ev: Dict, name: str) -> None:
    """``got`` (``[heads, n, D]``) within the bound of ``ev[name]``."""
    err = (got.double().cpu() - ev[name]).abs()
    worst = (err / ev["bound"][name]).max().item()
    assert worst <= 1.0, f"{name}: error {worst:.2f} times its bound"
