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


# ---- fp16 gradients far from one ------------------------------------------------------------------------------------------
def gradients(q, k, v, d_o, scale, causal=False, lengths=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    got = torch.autograd.grad(na.attention(q, k, v, scale, causal, lengths), (q, k, v), d_o)
    na.check_kernels(DEV)
    return got


def near(got, want, terms, units, what):
    """`units` roundings of fp16 in the norm, of the gradient or, where its terms cancel, of these; and half a step of the
    numbers below 2^-14, which are 2^-24 apart."""
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - want).square().mean().sqrt()
    bound = units * U[F16] * want.square().mean().sqrt().clamp_min(terms) + 2.0 ** -25
    assert err <= bound, f"{what}: {err:.2e} of {bound:.2e}"


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 100.0])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("C,Tq,Tk", [(128, 600, 8192), (64, 130, 16384), (128, 4096, 4096)])
def test_fp16_gradients_of_any_size_on_long_rows(C, Tq, Tk, causal, size):
    """Weights of 2^-14 times gradients of 1e-4 are below every number of fp16.  K is large for dq and Q for dk, so that the results
    themselves are not."""
    for name, kq in (("dq", (1 / 64, 64.0)), ("dk", (64.0, 1 / 64))):
        q, k = rand(1, 2, Tq, C, dtype=F16, scale=kq[0]), rand(1, 1, Tk, C, dtype=F16, seed=1, scale=kq[1])
        v, d_o = rand(1, 1, Tk, C, dtype=F16, seed=2), rand(1, 2, Tq, C, dtype=F16, seed=3, scale=size)
        got = gradients(q, k, v, d_o, C ** -0.5, causal)
        want = plain_attention(q, k, v, d_o, C ** -0.5, causal, None)
        if name == "dq":
            near(got[0], want[2], want[5][0], 1.5, name)
        else:
            near(got[1], want[3], want[6][0], 1.5, name)
        near(got[2], want[4], 0.0, 1.5, "dv")


@pytest.mark.parametrize("N,Nk,Tq,Tk,C", [(2, 2, 200, 40, 64), (4, 2, 30, 150, 128), (2, 1, 1000, 100, 32)])
def test_fp16_gradients_that_are_large_on_the_way(N, Nk, Tq, Tk, C):
    """dO . V reaches 1e7, dq and dk do not."""
    q, k = rand(1, N, Tq, C, dtype=F16, scale=0.01), rand(1, Nk, Tk, C, dtype=F16, seed=1, scale=0.01)
    v, d_o = rand(1, Nk, Tk, C, dtype=F16, seed=2, scale=30.0), rand(1, N, Tq, C, dtype=F16, seed=3, scale=1e4)
    got = gradients(q, k, v, d_o, C ** -0.5)
    want = plain_attention(q, k, v, d_o, C ** -0.5, False, None)
    assert max(t.abs().max() for t in want[2:5]) < 65504
    near(got[0], want[2], want[5][0], 1.5, "dq")
    near(got[1], want[3], want[6][0], 1.5, "dk")
    near(got[2], want[4], 0.0, 1.5, "dv")


@pytest.mark.parametrize("C,Tq,Tk", [(128, 512, 8192), (64, 2000, 2000)])
def test_fp16_rows_of_different_sizes(C, Tq, Tk):
    """Every row's dq is as near as its own gradient allows, whatever the other rows' are."""
    size = torch.logspace(-5, 0, 8, device=DEV).repeat_interleave(Tq // 8)[:, None]
    q, k, v = rand(1, 1, Tq, C, dtype=F16, scale=1 / 64), rand(1, 1, Tk, C, dtype=F16, seed=1, scale=64.0), rand(1, 1, Tk, C, dtype=F16, seed=2)
    d_o = (rand(1, 1, Tq, C, seed=3) * size).to(F16)
    got = gradients(q, k, v, d_o, C ** -0.5)
    want = plain_attention(q, k, v, d_o, C ** -0.5, False, None)
    for i in range(8):
        rows = slice(i * (Tq // 8), (i + 1) * (Tq // 8))
        part = plain_attention(q[:, :, rows], k, v, d_o[:, :, rows], C ** -0.5, False, None)
        near(got[0][:, :, rows], part[2], part[5][0], 1.5, f"rows {i}")
    near(got[1], want[3], want[6][0], 1.5, "dk")


def test_fp16_gradients_without_a_workspace():
    """The C entry keeps its bounds elsewhere then; the gradients are the same sums (parts are joined in another order, then one rounding)."""
    B, N, Nk, Tq, Tk, C = 2, 4, 2, 300, 2100, 64
    q, k, v = rand(B, N, Tq, C, dtype=F16), rand(B, Nk, Tk, C, dtype=F16, seed=1), rand(B, Nk, Tk, C, dtype=F16, seed=2)
    d_o, lengths = rand(B, N, Tq, C, dtype=F16, seed=3, scale=1e-3), torch.tensor([2100, 77], device=DEV, dtype=torch.int32)
    o, lse = na.attention_with_lse(q, k, v, 0.125, False, lengths)
    want = plain_attention(q, k, v, d_o, 0.125, False, lengths)
    a, delta = _lib.AttentionArgs(), torch.empty_like(lse)
    a.struct_size = ctypes.sizeof(a)
    a.B, a.N, a.Nk, a.Tq, a.Tk, a.C, a.dtype, a.scale = B, N, Nk, Tq, Tk, C, _lib.DTYPE_F16, 0.125
    a.stream, a.lse, a.delta, a.key_lengths = torch.cuda.current_stream().cuda_stream, lse.data_ptr(), delta.data_ptr(), lengths.data_ptr()
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o), ("d_o", d_o)):
        setattr(a, name, _lib.Heads(t.data_ptr(), 0, 0, 0))
    for halves in ("qkv", "q", "kv"):
        out = {name: torch.full_like(t, math.nan) for name, t in (("q", q), ("k", k), ("v", v))}
        for name, t in out.items():
            setattr(a, "d_" + name, _lib.Heads(t.data_ptr() if name in halves else None, 0, 0, 0))
        room = _lib.lib.na2d_attention_workspace(ctypes.byref(a), 1)
        bounds = 4 * (B * N * Tq + 2 * B * Nk)
        assert room >= bounds
        workspace = torch.full((room,), 255, dtype=torch.uint8, device=DEV)
        for size in (0, bounds - 4, bounds + 64, room):
            a.workspace, a.workspace_bytes = (workspace.data_ptr(), size) if size else (None, 0)
            _lib.check(_lib.lib.na2d_attention_backward(ctypes.byref(a)))
            na.check_kernels(DEV)
            for b in range(B):
                for name, ref, terms in (("q", want[2], want[5]), ("k", want[3], want[6]), ("v", want[4], torch.zeros(B))):
                    if name in halves:
                        near(out[name][b], ref[b], float(terms[b]), 1.5, f"d{name} {b} {size}")


# ---- sums over very many pixels ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,groups,shift", [((1, 256, 256, 1028), 1, 0.0), ((1, 256, 256, 1028), 1, 300.0), ((1, 300, 333, 301), 1, 0.0)], ids=str)
def test_group_norm_of_wide_groups_on_large_maps(shape, groups, shift):
    """A group's values by the hundred thousand in one thread: the statistics are as near as the other forms'.  (With a mean of
    300 spreads x - mean itself is exact to 1.8e-5, as in test_group_norm_far_from_zero.)"""
    C = shape[-1]
    x, d_y = rand(*shape, shift=shift), rand(*shape, seed=3) + 0.5
    if shift:
        check_norm(x, groups, None, None, d_y, None, units=8)
    else:
        check_norm(x, groups, rand(C, seed=1, scale=0.3, shift=1.0), rand(C, seed=2), d_y)


# ---- waits that gave up ---------------------------------------------------------------------------------------------
def test_group_norm_raises_what_an_earlier_wait_reported():
    """Its kernels of two passes wait for one another; one that gave up wrote wrong values, and the next call, forward or backward, says so."""
    na.check_kernels(DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    x = rand(1, 4, 4, 8).requires_grad_()
    y = na.group_norm(x, 2)
    for call in (lambda: na.group_norm(x.detach(), 2), lambda: na.group_norm(x, 2), lambda: torch.autograd.grad(y, x, y.detach(), retain_graph=True)):
        _lib.check(_lib.lib.na2d_selftest_wait_timeout(0, stream, 1000))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bounded wait"):
            call()
        call()
    na.check_kernels(DEV)


# ---- not finite beside what sees nothing ---------------------------------------------------------------------------------
FORMS = [(F32, 32), (F32, 200), (BF16, 7), (BF16, 64), (F16, 128)]


@pytest.mark.parametrize("Tq", [7, 150])
@pytest.mark.parametrize("dtype,C", FORMS)
def test_rows_that_see_nothing_beside_infinite_keys(dtype, C, Tq):
    """o = 0 and dq = 0, although a visible key of their tile has a value that is not finite."""
    q, k, v = rand(1, 2, Tq, C, dtype=dtype), rand(1, 1, 40, C, dtype=dtype, seed=1), rand(1, 1, 40, C, dtype=dtype, seed=2)
    k[0, 0, 1, 0], v[0, 0, 0, 1], v[0, 0, 1, 2] = math.inf, math.inf, math.nan
    lengths = torch.tensor([3], device=DEV)                       # the last three rows see keys
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o, lse = na.attention_with_lse(q, k, v, 0.25, True, lengths)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
    assert (o[:, :, :Tq - 3] == 0).all() and (lse[:, :, :Tq - 3] == -math.inf).all()
    assert (dq[:, :, :Tq - 3] == 0).all()


@pytest.mark.parametrize("Tq", [3, 40])
@pytest.mark.parametrize("dtype,C", FORMS)
def test_tokens_that_see_nothing_beside_infinite_keys(dtype, C, Tq):
    """The form of serving, caches of different lengths."""
    q, k, v = rand(3, 4, Tq, C, dtype=dtype), rand(3, 2, 300, C, dtype=dtype, seed=1), rand(3, 2, 300, C, dtype=dtype, seed=2)
    k[:, :, 0, 0], v[:, :, 0, 1] = math.inf, math.inf
    lengths = torch.tensor([1, 0, 300], device=DEV)
    with torch.no_grad():
        o, lse = na.attention_with_lse(q, k, v, 0.25, True, lengths)
    for b, blind in enumerate((Tq - 1, Tq, 0)):
        assert (o[b, :, :blind] == 0).all() and (lse[b, :, :blind] == -math.inf).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,C", FORMS)
@pytest.mark.parametrize("B,N,Nk,Tq,Tk", [(1, 2, 1, 20, 90), (1, 2, 2, 1100, 200), (2, 4, 2, 9, 300)])
def test_keys_beyond_a_length_beside_infinite_gradients(B, N, Nk, Tq, Tk, dtype, C, causal):
    """dk = 0 and dv = 0 there, although the queries and the gradients that meet their tile are not finite."""
    q, k, v = rand(B, N, Tq, C, dtype=dtype), rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    d_o = rand(B, N, Tq, C, dtype=dtype, seed=3)
    q[:, 0, Tq - 1, 0], d_o[:, 0, Tq - 2, 1], d_o[:, -1, Tq - 1, 3] = math.nan, math.inf, -math.inf
    lengths = torch.tensor([Tk - 70, 5][:B], device=DEV)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o = na.attention(q, k, v, 0.25, causal, lengths)
    _, dk, dv = torch.autograd.grad(o, (q, k, v), d_o)
    for b in range(B):
        assert (dk[b, :, lengths[b]:] == 0).all() and (dv[b, :, lengths[b]:] == 0).all()


# ---- group norm in several sets of units -----------------------------------------------------------------------------
SETS = [  # shape, groups, type: several sets of the two passes, several units a set, a last set of fewer, slabs of several entries
    ((9, 128, 128, 256), 8, F32), ((9, 128, 128, 256), 8, BF16), ((4, 256, 256, 256), 16, F32), ((4, 256, 256, 256), 16, F16),
    ((40, 100, 100, 64), 2, F32), ((40, 100, 100, 64), 2, BF16), ((5, 256, 257, 100), 5, F32), ((3, 300, 300, 384), 12, BF16), ((10, 64, 64, 1024), 2, F16),
]


@pytest.mark.parametrize("shape,groups,dtype", SETS, ids=str)
def test_group_norm_in_several_sets(shape, groups, dtype):
    """Blocks wait for one another, reuse the runs' places and add to their rows of channel sums: right, the same bits every time, and
    the same parameter gradients where d_x is not wanted."""
    gen = torch.Generator(DEV).manual_seed(7)
    normal = lambda *s: torch.randn(s, generator=gen, device=DEV)
    C = shape[-1]
    x, d_y = (normal(*shape) * 1.5 + normal(shape[0], 1, 1, C)).to(dtype), normal(*shape).to(dtype)
    w, b = normal(C) * 0.3 + 1, normal(C)
    check_norm(x, groups, w, b, d_y)

    def step(wanted):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        y = na.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu")
        return [y.detach()] + list(torch.autograd.grad(y, [leaves[i] for i in wanted], d_y))
    first = step((0, 1, 2))
    for _ in range(3):
        same(step((0, 1, 2)), first)
    same(step((1, 2)), [first[0]] + first[2:])
    same(step((0,)), first[:2])
    na.check_kernels(DEV)


# ---- graphs ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["norm", "attention", "tokens", "rotary"])
def test_calls_in_a_graph(which):
    """Captured once, replayed on other values: the cooperative launch and its cleared counts, fp16's norms, parts of caches."""
    table = na.rotary_table(torch.arange(50, device=DEV), na.rotary_frequencies(32))
    shapes, call = {
        "norm": (((9, 128, 128, 128), (128,), (128,)), lambda x, w, b: na.group_norm(x, 8, w, b, activation="silu")),
        "attention": (((2, 4, 150, 64), (2, 2, 700, 64), (2, 2, 700, 64)), lambda q, k, v: na.attention(q.half(), k.half(), v.half(), 0.125)),
        "tokens": (((5, 8, 1, 64), (5, 4, 900, 64), (5, 4, 900, 64)),
                   lambda q, k, v: na.attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), 0.125, True, torch.arange(5, device=DEV) * 200)),
        "rotary": (((2, 3, 50, 32), (2, 1, 50, 32)), lambda q, k: torch.cat(na.rotary(q, k, table), 1)),
    }[which]
    inputs = [torch.randn(s, device=DEV).requires_grad_() for s in shapes]

    def step():
        y = call(*inputs)
        return [y, *torch.autograd.grad(y, inputs, torch.ones_like(y))] if which != "tokens" else [y]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.set_grad_enabled(which != "tokens"):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.set_grad_enabled(which != "tokens"):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            for t in inputs:
                t.normal_()
        graph.replay()
        got = [t.detach().clone() for t in out]
        with torch.set_grad_enabled(which != "tokens"):
            same(got, [t.detach() for t in step()])
    na.check_kernels(DEV)


# ---- sizes of serving --------------------------------------------------------------------------------------------------------
def check_tokens(B, N, Nk, Tq, Tk, C, dtype, lengths=None):
    q, k, v = rand(B, N, Tq, C, dtype=dtype), rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    lengths = None if lengths is None else torch.tensor(lengths, device=DEV)
    with torch.no_grad():
        o, lse = na.attention_with_lse(q, k, v, C ** -0.5, True, lengths)
    na.check_kernels(DEV)
    want = plain_attention(q, k, v, q, C ** -0.5, True, lengths)
    close(o, want[0], dtype, 1, "o")
    seen = want[1] > -math.inf
    assert torch.equal(lse == -math.inf, ~seen) and (lse.double() - want[1])[seen].abs().max() < 1e-4


@pytest.mark.parametrize("dtype,C", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("B,N,Nk,Tq", [(37, 8, 8, 1), (36, 8, 8, 1), (20, 32, 16, 1), (37, 16, 8, 5), (38, 32, 8, 9)])
def test_tokens_of_many_units(B, N, Nk, Tq, dtype, C):
    """On both sides of the number of units from which they are items by themselves."""
    check_tokens(B, N, Nk, Tq, 333, C, dtype, [333 * b // (B - 1) for b in range(B)])
    check_tokens(B, N, Nk, Tq, 260, C, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [6, 7, 8, 9, 16])
def test_tokens_of_as_many_heads_as_three_stages_take(G, dtype):
    check_tokens(2, 2 * G, 2, 1, 1500, 128, dtype, [1500, 700])


@pytest.mark.parametrize("N,Nk,Tq,C", [(4, 2, 1, 64), (2, 2, 2, 128), (6, 1, 1, 40)])
def test_tokens_in_32_bits_on_long_caches(N, Nk, Tq, C):
    check_tokens(2, N, Nk, Tq, 20000, C, F32, [20000, 4097])


# ---- fp16 weights far below the largest ------------------------------------------------------------------------------------
@pytest.mark.parametrize("below", [22.0, 24.5, 26.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,Tq,Tk,C", [(1, 1, 131072, 64), (2, 3, 65536, 128), (1, 40, 65536, 64), (1, 300, 32768, 128)])
def test_many_keys_of_small_weight_beside_one_of_large(N, Tq, Tk, C, dtype, below):
    """One key has nearly all weight and a value of zero; the others, 2^-below of it each, and a spread about that, make up the
    result.  Rounding them is unbiased as long as they are numbers of the type: one rounding's bound."""
    q, k = rand(1, N, Tq, C, dtype=dtype), rand(1, 1, Tk, C, dtype=dtype, seed=1, scale=0.3)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, :, 0] = 0.0
    k[:, :, 0, 0] = 16.0
    scale = below * math.log(2.0) / 128
    v = rand(1, 1, Tk, C, dtype=dtype, seed=2, scale=300.0, shift=1000.0)
    v[:, :, 0] = 0.0
    with torch.no_grad():
        o, lse = na.attention_with_lse(q, k, v, scale)
    na.check_kernels(DEV)
    want = plain_attention(q, k, v, q, scale, False, None)
    close(o, want[0], dtype, 1, "o")
    assert (lse.double() - want[1]).abs().max() < 1e-4
