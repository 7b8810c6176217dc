"""What autograd must see of the grouped-head attention and rotary calls, on
the CPU: the launch is replaced by one that fills the outputs with ones."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from flash_spacetime import (_lib, flash_grouped_attention, flash_grouped_attention_varlen,
                             flash_rotary, flash_rotary_varlen, grouped, rotary)

FREQS = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64)
CU = torch.tensor([0, 4, 6], dtype=torch.int32)


@pytest.fixture
def launches(monkeypatch):
    """Entry points called, in order."""
    names = []

    def ones(rows, count):
        if rows.data:
            (ctypes.c_float * count).from_address(rows.data)[:] = [1.0] * count

    def call(name, args, device):
        names.append(name)
        if name == "fst_grouped_forward":
            a = _lib.FstGroupedForwardArgs.from_buffer_copy(args)
            ones(a.out, a.prob.total_rows * a.prob.heads * a.prob.head_dim)
        elif name == "fst_rotary":
            a = _lib.FstRotaryArgs.from_buffer_copy(args)
            ones(a.q_out, a.total_rows * a.heads * a.head_dim)
            ones(a.k_out, a.total_rows * a.kv_heads * a.head_dim)

    for module in (grouped, rotary):
        monkeypatch.setattr(module, "_call", call)
        monkeypatch.setattr(module, "_check_tensor", lambda *_: None)
    return names


CALLS = [
    lambda q, k: flash_grouped_attention_varlen(q, k, k, CU),
    lambda q, k: flash_grouped_attention(q[None], k[None], k[None], [6], layout="blhd"),
    lambda q, k: flash_rotary_varlen(q, k, FREQS, CU)[0],
    lambda q, k: flash_rotary(q[None], k[None], FREQS, layout="blhd")[1],
]


def _inputs():
    return torch.randn(6, 4, 8), torch.randn(6, 2, 8)


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("call", CALLS)
def test_forward_mode_is_refused(launches, call, which, grad_mode):
    t = list(_inputs())
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(*t)


@pytest.mark.parametrize("call", CALLS)
def test_function_transforms_are_refused(launches, call):
    q, k = _inputs()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: call(x, k), (q,), (torch.ones_like(q),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: call(x, k).sum())(q)


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("call", CALLS)
def test_a_trace_runs_the_call_or_is_refused(launches, call, grad_mode):
    with torch.set_grad_enabled(grad_mode):
        try:
            traced = torch.jit.trace(call, _inputs(), check_trace=False)
        except RuntimeError:
            return
        del launches[:]
        out = traced(*_inputs())
    assert len(launches) == 1 and torch.equal(out, torch.ones_like(out))


@pytest.mark.parametrize("call", CALLS)
def test_other_calls_have_a_node_only_for_a_gradient(launches, call):
    q, k = _inputs()
    assert call(q, k).grad_fn is None
    assert call(q, k.requires_grad_(True)).requires_grad
    with torch.no_grad():
        assert not call(q, k).requires_grad
    assert len(launches) == 3
