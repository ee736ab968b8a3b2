"""group_norm, rotary and attention where a call is more than its kernels: saved tensors that hooks hand back, recorded calls, waits
that gave up, values that are not finite beside rows and keys that see nothing, gradients far from one, very long sums."""
import ctypes
import math

import pytest
import torch

import e_natten_b200 as na
from e_natten_b200 import _lib
from test_gpu_block import BF16, F16, F32, U, check_norm, close, plain_attention, rand

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---- saved tensors and gradients of another form ----------------------------------------------------------------
def refused_in_backward(call, leaves, change, which):
    """The backward of call() is refused where hooks hand back change(t) for the saved tensors that `which` picks."""
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if which(t) else t):
        out = call()
    out = [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
    before = na.launch_count()
    with pytest.raises((ValueError, RuntimeError)):
        torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])
    assert na.launch_count() == before


CHANGES = {"cpu": lambda t: t.cpu(), "row": lambda t: t[:1], "half": lambda t: t.half(), "dims": lambda t: t.unsqueeze(0),
           "short": lambda t: t.flatten()[:1]}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("which", ["table", "index"])
def test_rotary_refuses_saved_tensors_of_another_form(change, which):
    table = na.rotary_table(torch.arange(9, device=DEV), na.rotary_frequencies(32))
    index = torch.arange(8, device=DEV).view(2, 4)
    q, k = rand(2, 3, 4, 32).requires_grad_(), rand(2, 1, 4, 32, seed=1).requires_grad_()
    if which == "table" and change == "row":
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1] if t.is_floating_point() else t):
            out = na.rotary(q, k, table, index)     # a shorter table is a table: the rows that it lacks are NaN
        gq, gk = torch.autograd.grad(out, (q, k), [torch.ones_like(t) for t in out])
        assert torch.isnan(gq[1]).all() and not torch.isnan(gq[0, :, 0]).any()
        return
    refused_in_backward(lambda: na.rotary(q, k, table, index), (q, k), CHANGES[change],
                        lambda t: t.is_floating_point() == (which == "table"))


def test_rotary_without_index_refuses_a_saved_table_of_too_few_rows():
    table = na.rotary_table(torch.arange(4, device=DEV), na.rotary_frequencies(32))
    q = rand(2, 3, 4, 32).requires_grad_()
    refused_in_backward(lambda: na.rotary(q, None, table), (q,), CHANGES["row"], lambda t: True)


@pytest.mark.parametrize("change", CHANGES)
def test_attention_refuses_saved_lengths_of_another_form(change):
    lengths = torch.tensor([5, 7], device=DEV, dtype=torch.int32)
    q, k, v = (rand(2, 2, 7, 32, dtype=BF16, seed=i).requires_grad_() for i in range(3))
    refused_in_backward(lambda: na.attention(q, k, v, key_lengths=lengths), (q, k, v), CHANGES[change], lambda t: not t.is_floating_point())


def test_a_lazily_negated_gradient_is_refused():
    """Its memory has the other sign."""
    x = rand(1, 2, 8, 32).requires_grad_()
    table = na.rotary_table(torch.arange(8, device=DEV), na.rotary_frequencies(32))
    for call in (lambda: na.rotary(x, None, table)[0], lambda: na.rotary(x, x, table)[1], lambda: na.attention(x, x, x), lambda: na.group_norm(x, 4)):
        y = call()
        with pytest.raises(ValueError, match="lazily negated"):
            torch.autograd.grad(y, x, torch._neg_view(torch.ones_like(y)))


def test_lazily_negated_tables_lengths_and_parameters_are_refused():
    x, negated = rand(2, 2, 8, 32), torch._neg_view
    table, index = na.rotary_table(torch.arange(8, device=DEV), na.rotary_frequencies(32)), torch.arange(16, device=DEV).view(2, 8) % 8
    lengths, w = torch.tensor([3, 5], device=DEV), rand(32)
    for call in (lambda: na.rotary(x, None, negated(table)), lambda: na.rotary(x, None, table, negated(index)),
                 lambda: na.attention(x, x, x, key_lengths=negated(lengths)), lambda: na.attention(x, x, x, key_lengths=negated(lengths.int())),
                 lambda: na.group_norm(x, 4, negated(w)), lambda: na.group_norm(x, 4, None, negated(w)),
                 lambda: na.rotary(negated(x), None, table), lambda: na.attention(x, negated(x), x), lambda: na.group_norm(negated(x), 4)):
        with pytest.raises(ValueError, match="lazily negated"):
            call()


def test_a_rotary_table_of_lazily_negated_positions():
    positions, frequencies = torch.arange(5, device=DEV, dtype=torch.float64), na.rotary_frequencies(8)
    want = na.rotary_table(-positions, -frequencies)
    assert torch.equal(na.rotary_table(torch._neg_view(positions), torch._neg_view(frequencies)), want)
