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


# ---- recorded calls -------------------------------------------------------------------------------------------------
def recorded(which):
    """(function of tensors, a maker of its arguments by seed)."""
    table = na.rotary_table(torch.arange(64, device=DEV), na.rotary_frequencies(32))
    grid = lambda seed: rand(2, 6, 7, 3, 4, 32, seed=seed).permute(3, 0, 4, 1, 2, 5).unbind(0)
    heads = lambda seed: (rand(2, 4, 9, 32, seed=seed), rand(2, 2, 40, 32, seed=seed + 1), rand(2, 2, 40, 32, seed=seed + 2))
    lengths = lambda seed: torch.tensor([40 - seed, 3 + seed], device=DEV)
    index = lambda seed: (torch.arange(18, device=DEV).view(2, 9) * (seed + 1)) % 64
    return {
        "attention": (lambda q, k, v, n: na.attention(q, k, v, 0.25, True, n), lambda s: (*heads(s), lengths(s))),
        "attention_bf16": (lambda q, k, v: na.attention(q, k, v, 0.25), lambda s: tuple(t.to(BF16) for t in heads(s))),
        "attention_with_lse": (lambda q, k, v: na.attention_with_lse(q, k, v, 0.25), heads),
        "attention_on_a_grid": (lambda q, k, v: na.attention(q, k, v, 0.25), grid),
        "group_norm": (lambda x, w, b: na.group_norm(x, 4, w, b, activation="silu"), lambda s: (rand(2, 5, 6, 32, seed=s), rand(32, seed=s), rand(32, seed=s + 1))),
        "group_norm_alone": (lambda x: na.group_norm(x, 4), lambda s: (rand(2, 5, 6, 32, seed=s),)),
        "group_norm_bias": (lambda x, b: na.group_norm(x, 4, None, b), lambda s: (rand(2, 5, 6, 32, seed=s), rand(32, seed=s))),
        "rotary": (lambda q, k, i: na.rotary(q, k, table, i), lambda s: (rand(2, 4, 9, 32, seed=s), rand(2, 2, 9, 32, seed=s + 1), index(s))),
        "rotary_of_one": (lambda q: na.rotary(q, None, table, interleaved=True)[0], lambda s: (rand(2, 4, 9, 48, seed=s),)),
        "rotary_on_a_grid": (lambda q, k: na.rotary(q, k, table), lambda s: grid(s)[:2]),
        "rotary_table": (lambda p, f: na.rotary_table(p, f, 1.5), lambda s: (torch.arange(9, device=DEV) * (s + 1), na.rotary_frequencies(32, 100.0 + s))),
    }[which]


RECORDED = ["attention", "attention_bf16", "attention_with_lse", "attention_on_a_grid", "group_norm", "group_norm_alone", "group_norm_bias", "rotary",
            "rotary_of_one", "rotary_on_a_grid", "rotary_table"]


def results(f, args, grad):
    """Outputs of f, and with `grad` the gradients of the floating arguments."""
    args = [t.detach().requires_grad_(grad and t.is_floating_point()) for t in args]
    out = f(*args)
    out = list(out) if isinstance(out, (tuple, list)) else [out]
    if not grad:
        return out
    ends = [t for t in out if t.requires_grad]
    return [t.detach() for t in out] + list(torch.autograd.grad(ends, [t for t in args if t.requires_grad], [torch.cos(t.detach()) for t in ends]))


def same(got, want):
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which,grad", [(w, g) for w in RECORDED for g in (False, True) if w != "rotary_table" or not g])
def test_a_traced_call_runs_again(which, grad):
    """On other values than it was traced with, and with gradients."""
    f, make = recorded(which)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, make(0), check_trace=False)
        for seed in (1, 2, 3):      # (the executor looks at the first runs and rewrites what follows)
            same(results(traced, make(seed), grad), results(f, make(seed), grad))


@pytest.mark.parametrize("which", RECORDED)
def test_a_call_recorded_by_a_dispatch_mode_runs_again(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, make = recorded(which)
    for grad in (False, True)[:1 if which == "rotary_table" else 2]:
        graph = make_fx(lambda *args: results(f, args, grad))(*make(0))
        same(graph(*make(1)), results(f, make(1), grad))
