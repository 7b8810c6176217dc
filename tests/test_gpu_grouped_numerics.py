"""What rounding may not do to grouped-head attention: gradients that are
exactly zero, common offsets, and the range of 16-bit values."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime import flash_grouped_attention, flash_grouped_attention_varlen

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
