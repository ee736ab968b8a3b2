"""prefix_attention, beam_select and beam_reorder against plain implementations in 64 bits, at the sizes and masks where they can go
wrong, and their refusals.

Tolerances of prefix_attention are those of attention (test_gpu_block.py): its weights are rounded to 16 bits for their products, its
results once, and what is joined in between is fp32.  beam_select's words and parents are exact; a score is rounded to fp32 once, and
its logarithm of a sum is off by less than 2^-22: exponentials by 2^-22 of themselves, of either sign, in sums of many.  beam_reorder
moves bytes.
"""
import ctypes
import math

import pytest
import torch

import e_natten_b200 as na
from e_natten_b200 import _lib
from test_gpu_block import BF16, DEV, F16, F32, close, differences, rand

pytestmark = pytest.mark.gpu


# ---- attention over a prefix ------------------------------------------------------------------------------------
def plain(q, pk, pv, k, v, d_o, scale, causal, lengths, prefix_lengths):
    """o, lse, the gradients of q, pk, pv, k, v, and the rms of the root of the summed squares of dq's, dpk's and dk's terms, in 64
    bits, entry by entry over the keys that it sees, one behind the other."""
    B, N, Tq, C = q.shape
    S, Nk, P = pk.shape[:3]
    Tk = 0 if k is None else k.shape[2]
    q, pk, pv, g = (t.double() for t in (q, pk, pv, d_o))
    k, v = (t.double() if t is not None else q.new_zeros(B, Nk, 0, C) for t in (k, v))
    o, dq, dpk, dpv, dk, dv = (torch.zeros_like(t) for t in (q, q, pk, pv, k, v))
    lse = torch.full((B, N, Tq), -math.inf, dtype=torch.float64, device=q.device)
    squares = [torch.zeros_like(t) for t in (q, pk, k)]
    row = torch.arange(Tq, device=q.device)
    for b in range(B):
        s = b // (B // S)
        L = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        Lp = P if prefix_lengths is None else min(max(int(prefix_lengths[s]), 0), P)
        seen = (L - Tq + 1 + row).clamp(0, L) if causal else torch.full_like(row, L)
        mask = torch.cat((torch.ones(Tq, Lp, dtype=torch.bool, device=q.device), torch.arange(L, device=q.device) < seen[:, None]), 1)
        ok = mask.any(1)
        if not ok.any():
            continue
        for m in range(Nk):
            heads = slice(m * (N // Nk), (m + 1) * (N // Nk))
            kk, vv = torch.cat((pk[s, m, :Lp], k[b, m, :L])), torch.cat((pv[s, m, :Lp], v[b, m, :L]))
            x = (q[b, heads][:, ok] @ kk.T * scale).masked_fill(~mask[ok], -math.inf)
            p = torch.softmax(x, -1)
            gg = g[b, heads][:, ok]
            dp = gg @ vv.T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            lse[b, heads] = lse[b, heads].masked_scatter(ok, x.logsumexp(-1))
            o[b, heads, ok] = p @ vv
            dq[b, heads, ok] = ds @ kk
            by_key, by_value = (ds.transpose(1, 2) @ q[b, heads][:, ok]).sum(0), (p.transpose(1, 2) @ gg).sum(0)
            dpk[s, m, :Lp] += by_key[:Lp]
            dpv[s, m, :Lp] += by_value[:Lp]
            dk[b, m, :L] += by_key[Lp:]
            dv[b, m, :L] += by_value[Lp:]
            terms = (p * dp * scale).square()
            squares[0][b, heads, ok] = terms @ kk.square()
            of_keys = (terms.transpose(1, 2) @ q[b, heads][:, ok].square()).sum(0)
            squares[1][s, m, :Lp] += of_keys[:Lp]
            squares[2][b, m, :L] += of_keys[Lp:]
    return o, lse, dq, dpk, dpv, dk, dv, squares


def rms(t, dtype=F32):
    """Of squares.  fp16's numbers below 2^-14 are 2^-24 apart: half of that is the rounding of a value of 2^-14."""
    return (t.mean().sqrt() if t.numel() else t.new_zeros(())).clamp_min(2.0 ** -14 if dtype == F16 else 0.0)


def check(q, pk, pv, k, v, d_o, scale=None, causal=False, lengths=None, prefix_lengths=None, path="auto", train=True, what=""):
    dtype = q.dtype
    leaves = [None if t is None else t.detach().requires_grad_(train) for t in (q, pk, pv, k, v)]
    o, lse = na.prefix_attention_with_lse(*leaves, scale, causal, lengths, prefix_lengths, path)
    grads = torch.autograd.grad(o, [t for t in leaves if t is not None], d_o) if train else None
    na.check_kernels(DEV)
    *want, squares = plain(q, pk, pv, k, v, d_o, 1.0 if scale is None else scale, causal, lengths, prefix_lengths)
    seen = want[1] > -math.inf
    assert torch.equal(lse == -math.inf, ~seen), f"{what}: rows that see nothing"
    assert (o[~seen] == 0).all()
    if seen.any():
        close(o.detach()[seen], want[0][seen], dtype, 1, f"o {what}")
        assert (lse.double() - want[1])[seen].abs().max() < 1e-4, f"lse {what}"
    if not train:
        return o, lse
    assert (grads[0][~seen] == 0).all()
    B, S = len(q), len(pk)
    for b in range(B):
        rows = seen[b]
        if rows.any():
            close(grads[0][b][rows], want[2][b][rows], dtype, 1.5, f"dq {b} {what}", rms(squares[0][b][rows], dtype))
    for s in range(S):
        L = pk.shape[2] if prefix_lengths is None else min(max(int(prefix_lengths[s]), 0), pk.shape[2])
        close(grads[1][s, :, :L], want[3][s, :, :L], dtype, 1.5, f"dpk {s} {what}", rms(squares[1][s, :, :L], dtype))
        close(grads[2][s, :, :L], want[4][s, :, :L], dtype, 1.5, f"dpv {s} {what}", rms(want[4][:0], dtype))
        assert (grads[1][s, :, L:] == 0).all() and (grads[2][s, :, L:] == 0).all()
    for b in range(B if k is not None else 0):
        L = k.shape[2] if lengths is None else min(max(int(lengths[b]), 0), k.shape[2])
        close(grads[3][b, :, :L], want[5][b, :, :L], dtype, 1.5, f"dk {b} {what}", rms(squares[2][b, :, :L], dtype))
        close(grads[4][b, :, :L], want[6][b, :, :L], dtype, 1.5, f"dv {b} {what}", rms(want[6][:0], dtype))
        assert (grads[3][b, :, L:] == 0).all() and (grads[4][b, :, L:] == 0).all()
    return o.detach(), grads


def operands(S, A, N, Nk, P, Tq, Tk, C, dtype, seed=0):
    B = S * A
    own = (rand(B, Nk, Tk, C, dtype=dtype, seed=seed + 3), rand(B, Nk, Tk, C, dtype=dtype, seed=seed + 4)) if Tk else (None, None)
    return (rand(B, N, Tq, C, dtype=dtype, seed=seed), rand(S, Nk, P, C, dtype=dtype, seed=seed + 1), rand(S, Nk, P, C, dtype=dtype, seed=seed + 2), *own,
            rand(B, N, Tq, C, dtype=dtype, seed=seed + 5))


SHAPES = [  # S, A, N, Nk, P, Tq, Tk, C
    (1, 1, 1, 1, 1, 1, 1, 32), (1, 3, 2, 1, 5, 4, 4, 64), (2, 2, 4, 2, 256, 12, 12, 16), (1, 4, 4, 4, 300, 130, 130, 64), (2, 3, 2, 2, 129, 64, 70, 128),
    (1, 8, 8, 2, 1000, 40, 40, 128), (3, 1, 2, 2, 140, 33, 35, 96), (1, 5, 6, 3, 513, 7, 260, 48), (1, 2, 2, 2, 1500, 300, 0, 64), (4, 2, 3, 3, 77, 20, 0, 32),
    (1, 16, 2, 1, 2100, 96, 96, 64),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefix_attention(shape, dtype, causal):
    *x, d_o = operands(*shape, dtype)
    check(*x, d_o, shape[-1] ** -0.5, causal)


@pytest.mark.parametrize("dtype,C", [(BF16, 7), (F16, 36), (BF16, 136), (F32, 130), (F32, 7)])
def test_prefix_attention_head_dims_without_tensor_cores(dtype, C):
    *x, d_o = operands(2, 3, 4, 2, 66, 20, 21, C, dtype)
    check(*x, d_o, C ** -0.5, True, torch.tensor([21, 0, 3, 21, 20, 1], device=DEV), torch.tensor([66, 11], device=DEV))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,Nk,P,Tq,Tk,C", [(4, 2, 300, 70, 300, 64), (2, 2, 200, 130, 256, 128), (8, 2, 400, 5, 150, 32), (2, 1, 260, 1, 140, 64)])
def test_prefix_attention_lengths(N, Nk, P, Tq, Tk, C, dtype, causal):
    """Prompts and answers of every length at which a tile or a step can end, none among them; what lies beyond is not looked at."""
    lengths = torch.tensor([0, 1, 2, 15, 16, 17, 127, 128, 129, Tk - 1, Tk, Tk + 9, -3, 0, 5], device=DEV)
    prefix_lengths = torch.tensor([P, 0, 1, 128, P + 5], device=DEV)         # three entries each: entries without any key are in the second's
    *x, d_o = operands(5, 3, N, Nk, P, Tq, Tk, C, dtype)
    o, grads = check(*x, d_o, C ** -0.5, causal, lengths, prefix_lengths)
    beyond = (torch.arange(Tk, device=DEV) >= lengths[:, None])[:, None, :, None]
    beyond_prefix = (torch.arange(P, device=DEV) >= prefix_lengths[:, None])[:, None, :, None]
    q, pk, pv, k, v = x
    poisoned = [q, pk.masked_fill(beyond_prefix, math.nan), pv.masked_fill(beyond_prefix, math.inf), k.masked_fill(beyond, math.inf), v.masked_fill(beyond, math.nan)]
    leaves = [t.detach().requires_grad_() for t in poisoned]
    o2 = na.prefix_attention(*leaves, C ** -0.5, causal, lengths.int(), prefix_lengths.int())
    grads2 = torch.autograd.grad(o2, leaves, d_o)
    assert torch.equal(o2, o)
    for name, a, b in zip(("dq", "dpk", "dpv", "dk", "dv"), grads2, grads):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("S,A,N,Nk,P,Tq,Tk,C", [
    (1, 64, 8, 2, 3000, 1, 200, 128),       # the prompt's rows by the 128-row kernel, own keys by the kernel of few rows
    (16, 4, 16, 4, 1000, 1, 100, 128),      # both by the latter: 16 rows a prompt
    (3, 8, 8, 2, 2100, 1, 333, 64),         # 32 rows
    (2, 3, 4, 2, 5000, 5, 17, 128),         # 30 and 10 rows
    (1, 11, 4, 1, 700, 1, 0, 32),           # the prompt alone
    (2, 9, 4, 1, 700, 1, 0, 96),            # the prompt alone, 36 rows
    (1, 2, 16, 2, 260, 5, 400, 64),         # own rows by the 128-row kernel, 40 of them
    (1, 1, 8, 2, 9000, 1, 300, 48), (40, 1, 4, 4, 64, 1, 2000, 128), (1, 24, 16, 4, 1111, 5, 70, 64), (1, 1, 1, 1, 1, 1, 1, 8),
    (300, 2, 2, 2, 40, 1, 30, 32),          # many short units
    (1, 130, 1, 1, 30000, 1, 5, 64),        # 130 rows on one key head: parts
])
def test_prefix_attention_of_tokens(S, A, N, Nk, P, Tq, Tk, C, dtype):
    *x, d_o = operands(S, A, N, Nk, P, Tq, Tk, C, dtype)
    B = S * A
    check(*x, d_o, C ** -0.5, True, train=False)
    lengths = torch.tensor([Tk * b // max(B - 1, 1) for b in range(B)], device=DEV) if Tk else None
    check(*x, d_o, C ** -0.5, True, lengths, torch.tensor([P - P * s // S for s in range(S)], device=DEV, dtype=torch.int32), train=False)
    if Tk:
        none = torch.zeros(B, device=DEV, dtype=torch.int64)
        o, lse = check(*x, d_o, C ** -0.5, True, none, none[:S], train=False)
        assert (o == 0).all() and (lse == -math.inf).all()


def test_prefix_attention_of_more_entries_than_the_line_takes():
    *x, d_o = operands(1, 4200, 1, 1, 70, 1, 20, 32, BF16)
    check(*x, d_o, 32 ** -0.5, True, torch.arange(4200, device=DEV) % 21, train=False)


@pytest.mark.parametrize("Tq,N", [(1, 2), (6, 2), (40, 2)])
def test_prefix_attention_paths_agree(Tq, N):
    """The same call on tensor cores and on CUDA cores: roundings of P apart."""
    *x, d_o = operands(2, 4, N, 2, 500, Tq, 50, 64, BF16)
    got = [check(*x, d_o, 0.125, True, path=path)[0] for path in ("tensor", "simt")]
    close(got[0], got[1], BF16, 2, "paths")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Tq", [1, 9, 140])
def test_prefix_attention_on_views(dtype, Tq):
    """q, k, v of one projection, (whose rows of an entry follow the entry's before); caches with tokens first; a crop whose rows do not
    follow; a prefix cut out of a longer cache; gradients with heads last."""
    S, A, N, C, P = 2, 3, 4, 64, 150
    B = S * A
    packed = rand(B, Tq, 3, N, C, dtype=dtype).permute(2, 0, 3, 1, 4)
    pk, pv = (rand(S, P + 9, 2, N, C, dtype=dtype, seed=1)[:, 3:P + 3].permute(2, 0, 3, 1, 4))
    d_o = rand(B, Tq, N, C, dtype=dtype, seed=2).permute(0, 2, 1, 3)
    crop = rand(B, N + 1, Tq + 5, C, dtype=dtype, seed=3)[:, 1:, 2:Tq + 2]
    odd = rand(B, N, Tq, C + 8, dtype=dtype, seed=4)[..., 8:]
    for q in (packed[0], crop, odd):
        check(q, pk, pv, packed[1], packed[2], d_o, 0.125, True)
    check(packed[0], pk, pv, crop, odd, d_o, 0.125, False)
    expanded = pk[:1].expand(S, -1, -1, -1)
    check(crop, expanded, pv, None, None, d_o, 0.125)


def test_prefix_attention_on_grids():
    S, A, H, W, N, C = 1, 2, 5, 7, 2, 32
    q, k, v, d_o = (rand(S * A, N, H, W, C, dtype=BF16, seed=i) for i in range(4))
    pk, pv = rand(S, N, 9, 11, C, dtype=BF16, seed=5), rand(S, N, 9, 11, C, dtype=BF16, seed=6)
    leaves = [t.requires_grad_() for t in (q, pk, pv, k, v)]
    o, lse = na.prefix_attention_with_lse(*leaves, 0.2)
    assert o.shape == q.shape and lse.shape == q.shape[:-1]
    grads = torch.autograd.grad(o, leaves, d_o)
    flat = [t.detach().flatten(2, 3) for t in leaves]
    want, want_grads = check(*flat, d_o.flatten(2, 3), 0.2)
    assert torch.equal(o.detach().flatten(2, 3), want)
    for a, b in zip(grads, want_grads):
        assert torch.equal(a.flatten(2, 3), b)


def test_prefix_attention_is_attention_over_both():
    """Against the operator beside it, on keys put behind one another: two roundings of each."""
    S, A, N, Nk, P, T, C = 2, 3, 4, 2, 200, 60, 64
    *x, d_o = operands(S, A, N, Nk, P, T, T, C, BF16)
    q, pk, pv, k, v = x
    both = [torch.cat((p.repeat_interleave(A, 0), own), 2) for p, own in ((pk, k), (pv, v))]
    close(na.prefix_attention(*x, 0.125), na.attention(q, *both, 0.125), BF16, 2, "not causal")
    close(na.prefix_attention(*x, 0.125, causal=True), na.attention(q, *both, 0.125, causal=True), BF16, 2, "causal")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,N,P,Tq,Tk", [(0, 2, 4, 4, 4), (2, 0, 4, 4, 4), (2, 2, 4, 0, 4), (2, 2, 0, 4, 0), (2, 2, 0, 4, 5), (2, 2, 5, 4, 0)])
def test_prefix_attention_of_nothing(B, N, P, Tq, Tk, dtype):
    q = rand(max(B, 1), max(N, 1), max(Tq, 1), 32, dtype=dtype)[:B, :N, :Tq].contiguous()
    pk, pv = (rand(1, 1, P, 32, dtype=dtype, seed=i) for i in (1, 2))
    k, v = (rand(max(B, 1), 1, Tk, 32, dtype=dtype, seed=i)[:B] for i in (3, 4))
    leaves = [t.detach().requires_grad_() for t in (q, pk, pv, k, v)]
    o, lse = na.prefix_attention_with_lse(*leaves)
    d_o = torch.ones_like(o)
    grads = torch.autograd.grad(o, leaves, d_o)
    for t, g in zip(leaves, grads):
        assert g.shape == t.shape
    *want, squares = plain(q, pk, pv, k, v, d_o, 1.0, False, None, None)
    assert o.shape == q.shape
    if o.numel():
        close(o.detach(), want[0], dtype, 1, "o")
        for g, ref, terms in zip(grads, want[2:7], (squares[0], squares[1], None, squares[2], None)):
            close(g, ref, dtype, 1.5, "gradient", 0.0 if terms is None else rms(terms))


def test_prefix_attention_is_the_same_every_time_and_on_any_stream():
    *x, d_o = operands(2, 4, 8, 2, 900, 50, 60, 64, F16)
    tokens = operands(2, 8, 8, 2, 900, 1, 60, 64, F16)[:5]

    def step():
        leaves = [t.detach().requires_grad_() for t in x]
        o = na.prefix_attention(*leaves, 0.125, True)
        with torch.no_grad():
            return (o.detach(), *torch.autograd.grad(o, leaves, d_o), na.prefix_attention(*tokens, 0.125, True))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_prefix_attention_needs_only_some_gradients():
    *x, d_o = operands(2, 3, 4, 2, 200, 33, 40, 64, BF16)
    whole = [t.detach().requires_grad_() for t in x]
    want = torch.autograd.grad(na.prefix_attention(*whole, 0.125, True), whole, d_o)
    for i in range(5):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(x)]
        got, = torch.autograd.grad(na.prefix_attention(*some, 0.125, True), some[i], d_o)
        assert torch.equal(got, want[i])
    some = [t.detach().requires_grad_(j == 2) for j, t in enumerate(x[:3])]
    got, = torch.autograd.grad(na.prefix_attention(*some, None, None, 0.125), some[2], d_o)
    whole = [t.detach().requires_grad_() for t in x[:3]]
    assert torch.equal(got, torch.autograd.grad(na.prefix_attention(*whole, scale=0.125), whole, d_o)[2])


def test_prefix_attention_gradient_against_differences():
    *x, d_o = operands(2, 2, 4, 2, 70, 10, 12, 16, F32)
    lengths, prefix_lengths = torch.tensor([12, 3, 12, 10], device=DEV), torch.tensor([66, 13], device=DEV)
    call = lambda: na.prefix_attention(*x, 0.25, True, lengths, prefix_lengths)
    leaves = [t.clone().requires_grad_() for t in x]
    grads = torch.autograd.grad(na.prefix_attention(*leaves, 0.25, True, lengths, prefix_lengths), leaves, d_o)
    with torch.no_grad():
        for t, g in zip(x, grads):
            entries = list(range(3, t.numel(), t.numel() // 12))
            # truncation h^2, rounding of the sum (about 1e-6) over 2 h
            got = differences(call, t, d_o, entries, 1e-2)
            assert (got - g.reshape(-1)[entries].double().cpu()).abs().max() < 2e-3


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefix_attention_joins_halves_of_any_weight(dtype):
    """Logits of the prompt far above, far below, and beside those of the own keys: e^(lse - lse) from 0 to 1."""
    *x, d_o = operands(1, 3, 2, 2, 100, 40, 40, 64, dtype)
    for by in (0.01, 1.0, 30.0):
        q, pk, pv, k, v = x
        check(q, (pk * by).to(dtype), pv, k, v, d_o, 0.125, True)
        check(q[:, :, :1].contiguous(), (pk * by).to(dtype), pv, k, v, d_o[:, :, :1].contiguous(), 0.125, True, train=False)


def test_prefix_attention_infinities_and_nan():
    """A NaN of one entry's query, and an infinite key of one prompt, reach their own rows only."""
    *x, d_o = operands(2, 2, 2, 2, 130, 3, 20, 64, BF16)
    q, pk, pv, k, v = x
    q[1, 0, 2] = math.nan
    pk[1, 1, 7, 0] = math.inf
    with torch.no_grad():
        o = na.prefix_attention(q, pk, pv, k, v, 0.125)
    bad = torch.isnan(o).any(-1)
    want = torch.zeros_like(bad)
    want[1, 0, 2] = True
    sign = q[2:, 1, :, 0].double() > 0                   # +infinity among the logits: NaN; -infinity: a weight of zero
    want[2:, 1] = sign
    assert torch.equal(bad, want)


@pytest.mark.parametrize("odd", [("o",), ("d_q",), ("d_k",), ("d_prefix_v",), ("o", "d_q", "d_k", "d_v", "d_prefix_k", "d_prefix_v")])
@pytest.mark.parametrize("dtype,C,Tq,Tk", [(F32, 32, 5, 7), (F32, 20, 1, 3), (BF16, 64, 40, 9), (BF16, 64, 1, 0), (F16, 20, 9, 7)])
def test_prefix_attention_results_on_any_place(dtype, C, Tq, Tk, odd):
    """Results of the C ABI that start one element behind a 16-byte boundary: what the same kernels write elsewhere, bit by bit, and
    nothing beside them."""
    B, S, N, Nk, P = 4, 2, 4, 2, 37
    q, d_o = rand(B, N, Tq, C, dtype=dtype), rand(B, N, Tq, C, dtype=dtype, seed=1)
    pk, pv = rand(S, Nk, P, C, dtype=dtype, seed=2), rand(S, Nk, P, C, dtype=dtype, seed=3)
    k, v = rand(B, Nk, Tk, C, dtype=dtype, seed=4), rand(B, Nk, Tk, C, dtype=dtype, seed=5)
    lse = torch.empty(B, N, Tq, device=DEV)

    def call(odd, forward, backward):
        a = _lib.PrefixAttentionArgs()
        a.struct_size = ctypes.sizeof(a)
        a.B, a.S, a.N, a.Nk, a.Tq, a.Tk, a.P, a.C = B, S, N, Nk, Tq, Tk, P, C
        a.dtype, a.scale = {F32: 0, BF16: 1, F16: 2}[dtype], 0.3
        a.stream = torch.cuda.current_stream(DEV).cuda_stream
        for name, t in (("q", q), ("prefix_k", pk), ("prefix_v", pv)) + ((("k", k), ("v", v)) if Tk else ()):
            setattr(a, name, _lib.Heads(t.data_ptr(), 0, 0, 0))
        a.lse = lse.data_ptr()
        out = {}

        def give(name, like):
            room = torch.full((like.numel() + 16,), 7.0, dtype=dtype, device=DEV)
            at = 1 if name in odd else 0
            out[name] = (room, room[at:at + like.numel()].view(like.shape))
            setattr(a, name, _lib.Heads(out[name][1].data_ptr(), 0, 0, 0))

        def run(path, of_backward):
            a.path = path
            need = _lib.lib.na2d_prefix_attention_workspace(ctypes.byref(a), of_backward)
            assert need > 0
            workspace = torch.empty(need, dtype=torch.uint8, device=DEV)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), need
            _lib.check((_lib.lib.na2d_prefix_attention_backward if of_backward else _lib.lib.na2d_prefix_attention_forward)(ctypes.byref(a)))
            na.check_kernels(DEV)

        give("o", q)
        run(forward, 0)
        a.d_o = _lib.Heads(d_o.data_ptr(), 0, 0, 0)
        for name, like in (("d_q", q), ("d_prefix_k", pk), ("d_prefix_v", pv)) + ((("d_k", k), ("d_v", v)) if Tk else ()):
            give(name, like)
        run(backward, 1)
        for name, (room, t) in out.items():
            at = 1 if name in odd else 0
            assert (room[:at] == 7).all() and (room[at + t.numel():] == 7).all(), name
        return {name: t for name, (_, t) in out.items()}

    # (o, and gradients of keys, that lie so are the CUDA cores'; a d_q is not)
    simt = _lib.PATH_SIMT
    forward = simt if "o" in odd else _lib.PATH_AUTO
    backward = _lib.PATH_AUTO if odd == ("d_q",) or not Tk and odd == ("d_k",) else simt
    want = call((), forward, backward)
    for name, t in call(odd, _lib.PATH_AUTO, _lib.PATH_AUTO).items():
        assert torch.equal(t, want[name]), name


@pytest.mark.parametrize("Tq", [1, 40])
def test_prefix_attention_in_a_graph(Tq):
    S, A, N, Nk, P, Tk, C = 2, 4, 4, 2, 600, 40, 64
    *x, d_o = operands(S, A, N, Nk, P, Tq, Tk, C, BF16)
    lengths, prefix_lengths = torch.full((S * A,), Tk, device=DEV, dtype=torch.int32), torch.full((S,), P, device=DEV, dtype=torch.int32)
    x = [t.requires_grad_(Tq > 1) for t in x]

    def step():
        o = na.prefix_attention(*x, 0.125, True, lengths, prefix_lengths)
        return [o.detach(), *torch.autograd.grad(o, x, d_o)] if Tq > 1 else [o]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            for t in x:
                t.normal_()
            lengths.copy_((torch.arange(S * A, device=DEV) * (i + 3)).clamp(max=Tk))
            prefix_lengths.copy_(torch.tensor([P - 31 * i, 200 * i], device=DEV))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    na.check_kernels(DEV)


# ---- beam search: the choice --------------------------------------------------------------------------------------
def plain_select(logits, scores, count, finished, end):
    """The whole line of every entry's candidates, sorted, in 64 bits."""
    B, K, V = logits.shape
    line = torch.log_softmax(logits.double(), -1) + scores.double()[..., None]
    bad = torch.isnan(logits).any(-1) | (logits == math.inf).any(-1) | ~torch.isfinite(scores)
    if finished is not None:
        itself = torch.full_like(line, -math.inf)
        itself[..., end] = scores.double()
        line = torch.where(finished[..., None], itself, line)
        bad = torch.where(finished, ~torch.isfinite(scores), bad)
    line = torch.where(bad[..., None] | torch.isnan(line), -math.inf, line).flatten(1)
    if line.shape[1] < count:
        line = torch.cat((line, line.new_full((B, count - line.shape[1]), -math.inf)), 1)
    found, at = torch.sort(line, dim=-1, descending=True, stable=True)
    found, at = found[:, :count], at[:, :count]
    at = torch.where(found > -math.inf, at, 0)
    return found, at // V, at % V


def check_select(logits, scores, count=None, finished=None, end=0):
    got = na.beam_select(logits, scores, count, finished, end)
    want = plain_select(logits, scores, logits.shape[1] if count is None else count, finished, end)
    assert got[0].dtype == F32 and got[1].dtype == got[2].dtype == torch.int64
    assert got[0].shape == got[1].shape == got[2].shape == want[0].shape
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    there = want[0] > -math.inf
    assert torch.equal(got[0] > -math.inf, there)
    # one rounding to fp32, and the logarithm of a sum off by 2^-22
    assert ((got[0].double() - want[0])[there].abs() <= 2.0 ** -24 * want[0][there].abs() + 2.0 ** -22).all()
    return got


def beams(B, K, V, dtype, seed=0, scale=3.0):
    return rand(B, K, V, dtype=F32, seed=seed, scale=scale).to(dtype), rand(B, K, seed=seed + 1, scale=2.0, shift=-9.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,K,V,count", [
    (1, 1, 1, 1), (2, 3, 2, 3), (4, 4, 16, 8), (1, 32, 17, 64), (3, 5, 255, 5), (2, 1, 4096, 1), (2, 4, 4097, 8), (5, 2, 8191, 4), (1, 4, 50021, 33),
    (2, 8, 65536, 16), (1, 1, 300007, 64), (70, 2, 1000, 2), (9, 16, 12289, 32), (1, 2, 5, 64), (300, 8, 4100, 8),
])
def test_beam_select(B, K, V, count, dtype):
    logits, scores = beams(B, K, V, dtype)
    check_select(logits, scores, count)
    finished = torch.rand(B, K, generator=torch.Generator().manual_seed(1)).to(DEV) < 0.4
    check_select(logits, scores, count, finished, V - 1)
    check_select(logits, scores)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_beam_select_of_equal_words(V, dtype):
    """All logits equal, few values, beams that are copies of one another: the lowest beam, then the lowest word."""
    scores = torch.full((2, 3), -1.5, device=DEV)
    same = torch.zeros(2, 3, V, device=DEV, dtype=dtype)
    parents, words = check_select(same, scores, 10)[1:]
    assert (parents == 0).all() and torch.equal(words, torch.arange(10, device=DEV).expand(2, 10))
    few = torch.randint(3, (2, 1, V), generator=torch.Generator().manual_seed(V)).to(DEV).to(dtype).expand(2, 3, V)
    check_select(few, scores, 10)
    check_select(few.contiguous(), scores, 64)
    copies = beams(2, 1, V, dtype)[0].expand(2, 3, V).contiguous()
    parents = check_select(copies, scores, 9)[1]
    if dtype == F32:                                     # (in 16 bits a beam's best words are often equal themselves)
        assert torch.equal(parents, torch.tensor([0, 1, 2], device=DEV).repeat(3).expand(2, 9))
    if dtype == F32:
        zeros = torch.zeros(1, 1, V, device=DEV)
        zeros[0, 0, 3] = -0.0                            # no less than the others
        assert check_select(zeros, scores[:1, :1], 5)[2].tolist() == [[0, 1, 2, 3, 4]]


@pytest.mark.parametrize("count", [1, 7, 33, 64])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_beam_select_of_sorted_words(count, dtype):
    """Ascending and descending logits: every word, and none, is better than those before it."""
    V = 30011 if dtype == F32 else 2000
    up = torch.linspace(-4, 4, V, device=DEV).to(dtype).expand(1, 2, V).contiguous()
    scores = torch.tensor([[-1.0, -1.25]], device=DEV)
    check_select(up, scores, count)
    check_select(up.flip(-1).contiguous(), scores, count)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [30, 9000])
def test_beam_select_of_words_that_are_ruled_out(V, dtype):
    logits, scores = beams(4, 3, V, dtype)
    logits[0] = -math.inf                                # no candidate at all
    logits[1, :, 5:] = -math.inf                         # five words are left
    logits[2, 1, 4] = math.nan
    logits[3, 0, 2] = math.inf
    logits[3, 1] = torch.finfo(dtype).min                # the type's lowest value is a value
    found, parents, words = check_select(logits, scores, 20)
    assert (found[0] == -math.inf).all() and (parents[0] == 0).all() and (words[0] == 0).all()
    assert (found[1, 15:] == -math.inf).all() and (found[1, :15] > -math.inf).all()
    assert not (parents[2] == 1).any() and not ((parents[3] == 0) & (found[3] > -math.inf)).any()
    scores[2, 0] = -math.inf
    scores[3, 2] = math.nan
    scores[1, 1] = math.inf
    check_select(logits, scores, 20)
    check_select(logits, scores, 20, torch.tensor([[True, False, True]], device=DEV).expand(4, 3), 7)
    check_select(logits, scores, 5, torch.ones(4, 3, dtype=torch.bool, device=DEV), 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_select_of_views(dtype):
    """The newest token's logits out of all tokens', rows that start anywhere, beams in another order, scores with strides."""
    K, V = 3, 5003
    every = rand(6, 4, V, dtype=F32, scale=3.0).to(dtype)
    scores = rand(K, 2, seed=1).t()
    check_select(every.view(2, 3, 4, V)[:, :, -1], scores, 6)
    check_select(rand(2, K, V + 9, dtype=F32, scale=3.0).to(dtype)[..., 5:V + 5], scores, 6)
    check_select(every[:, 0].view(K, 2, V).transpose(0, 1), scores, 6)
    check_select(rand(V, 2, K, dtype=F32, scale=3.0).to(dtype).permute(1, 2, 0), scores, 6)
    check_select(every[:1, :1].expand(2, K, V), scores, 6)


def test_beam_select_of_nothing_and_in_a_graph():
    got = na.beam_select(torch.zeros(0, 3, 5, device=DEV), torch.zeros(0, 3, device=DEV), 4)
    assert all(t.shape == (0, 4) for t in got)
    logits, scores = beams(3, 4, 20000, BF16)
    finished = torch.zeros(3, 4, dtype=torch.bool, device=DEV)
    na.beam_select(logits, scores, 8, finished, 3)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, count in zip(graphs, (8, 3)):
        with torch.cuda.graph(graph):
            outs.append(na.beam_select(logits, scores, count, finished, 3))
    for i in range(3):
        logits.normal_(std=3.0)
        scores.normal_()
        finished.bernoulli_(0.3)
        for j in (0, 1, 1, 0):
            graphs[j].replay()
        for out, count in zip(outs, (8, 3)):
            want = plain_select(logits, scores, count, finished, 3)
            assert torch.equal(out[1], want[1]) and torch.equal(out[2], want[2])


# ---- beam search: the caches --------------------------------------------------------------------------------------
def plain_reorder(cache, parents, lengths=None):
    B, K = parents.shape
    out = cache.clone()
    for e, p in enumerate(parents.flatten().tolist()):
        if 0 <= p < K:
            source = e // K * K + p
            if lengths is None:
                out[e] = cache[source]
            else:
                n = max(0, min(int(lengths.flatten()[source]), cache.shape[2]))
                out[e, :, :n] = cache[source, :, :n]
    return out


def bits(*shape, dtype=torch.uint8, seed=0):
    raw = torch.randint(0, 2 if dtype == torch.bool else 120, shape, generator=torch.Generator().manual_seed(seed + sum(shape)))
    return raw.to(dtype).to(DEV)


def parents_of(B, K, seed=0, index=torch.int64):
    return torch.randint(K, (B, K), generator=torch.Generator().manual_seed(seed)).to(index).to(DEV)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [F32, BF16, torch.int64, torch.uint8, torch.bool, torch.float8_e4m3fn])
@pytest.mark.parametrize("B,K,heads,T,C", [(1, 2, 1, 1, 1), (4, 4, 2, 12, 16), (3, 5, 3, 33, 7), (2, 8, 4, 100, 64), (1, 17, 2, 50, 48), (2, 32, 1, 9, 128), (5, 3, 2, 700, 40)])
def test_beam_reorder(B, K, heads, T, C, dtype, index):
    parents = parents_of(B, K, T, index)
    caches = [bits(B * K, heads, T, C, dtype=dtype, seed=i) for i in range(2)] + [bits(B * K, T, heads, C, dtype=dtype, seed=2).transpose(1, 2)]
    want = [plain_reorder(c, parents) for c in caches]
    na.beam_reorder(caches, parents)
    for got, ref in zip(caches, want):
        assert torch.equal(got.view(torch.uint8) if dtype == torch.float8_e4m3fn else got, ref.view(torch.uint8) if dtype == torch.float8_e4m3fn else ref)
    lengths = torch.randint(-1, T + 2, (B * K,), generator=torch.Generator().manual_seed(1)).to(index).to(DEV)
    caches = [bits(B * K, heads, T, C, dtype=torch.int32, seed=5), bits(B * K, T, heads, C, dtype=torch.int16, seed=6).transpose(1, 2)]
    want = [plain_reorder(c, parents, lengths) for c in caches]
    na.beam_reorder(caches, parents, lengths)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    cache = caches[0].clone()
    na.beam_reorder(cache, parents, lengths.view(B, K))
    assert torch.equal(cache, plain_reorder(caches[0], parents, lengths))


def test_beam_reorder_of_beams_that_stay_or_are_none():
    cache = bits(8, 2, 20, 16, dtype=torch.int32)
    was = cache.clone()
    stay = torch.arange(4, device=DEV).expand(2, 4)
    na.beam_reorder(cache, stay)
    assert torch.equal(cache, was)
    wild = torch.tensor([[1, -1, 4, 0], [7, 3, 2 ** 31 - 1, -2 ** 31]], device=DEV)
    want = plain_reorder(cache, wild)
    na.beam_reorder(cache, wild)
    assert torch.equal(cache, want)
    na.beam_reorder(cache, wild.int())
    far = torch.tensor([[2 ** 32, 2 ** 40 + 1, 1, -2 ** 33 + 2], [0, 0, 0, 0]], device=DEV)      # 64 bits, not their lower half
    want = plain_reorder(cache, far)
    na.beam_reorder(cache, far)
    assert torch.equal(cache, want)
    one = bits(3, 2, 5, 4)
    na.beam_reorder(one, torch.zeros(3, 1, dtype=torch.int64, device=DEV))
    assert torch.equal(one, bits(3, 2, 5, 4))


def test_beam_reorder_of_views():
    """Keys and values of one tensor, a cache given twice, caches cut out of larger ones (whose rest stays), states of other shapes."""
    B, K = 3, 4
    parents = parents_of(B, K, 7)
    whole = bits(B * K, 2, 3, 30, 32, dtype=torch.int16)
    was = whole.clone()
    na.beam_reorder([whole[:, 0], whole[:, 1]], parents)
    assert torch.equal(whole[:, 0], plain_reorder(was[:, 0], parents)) and torch.equal(whole[:, 1], plain_reorder(was[:, 1], parents))
    cache = bits(B * K, 3, 30, 32, dtype=torch.int16)
    want = plain_reorder(plain_reorder(cache, parents), parents)
    na.beam_reorder([cache, cache], parents)
    assert torch.equal(cache, want)
    large = bits(B * K + 2, 5, 40, 48, dtype=torch.int16)
    was, want = large.clone(), large.clone()
    cut = large[1:-1, 1:4, 3:33, 5:37]                   # rows that start on odd places
    want[1:-1, 1:4, 3:33, 5:37] = plain_reorder(was[1:-1, 1:4, 3:33, 5:37], parents)
    na.beam_reorder(cut, parents)
    assert torch.equal(large, want)
    shapes = [bits(B * K, 77, dtype=torch.int64, seed=1), bits(B * K, dtype=torch.int32, seed=2), bits(B * K, 3, 5, seed=3), bits(B * K, 2, 3, 4, 5, dtype=torch.bool, seed=4)]
    want = [plain_reorder(t, parents) for t in shapes]
    na.beam_reorder(shapes, parents)
    assert all(torch.equal(a, b) for a, b in zip(shapes, want))
    empty = torch.zeros(B * K, 2, 0, 8, device=DEV)
    na.beam_reorder([empty], parents)
    na.beam_reorder([], parents)
    none = torch.zeros(0, 2, 3, 4, device=DEV)
    na.beam_reorder(none, torch.zeros(0, 4, dtype=torch.int64, device=DEV))


def test_beam_reorder_of_many_caches():
    parents = parents_of(2, 3, 3)
    caches = [bits(6, 2, 5 + i % 7, 8 + 8 * (i % 3), dtype=torch.int16, seed=i) for i in range(150)]
    want = [plain_reorder(c, parents) for c in caches]
    na.beam_reorder(caches, parents)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_beam_reorder_of_a_long_cache():
    """More bytes than 32 bits count, at the far end too."""
    cache = torch.zeros(2, 1, 1 << 21, 1024, dtype=torch.int8, device=DEV)       # 2 GB an entry
    cache[1, 0, -1, -9:] = 7
    cache[1, 0, 5] = 3
    na.beam_reorder(cache, torch.tensor([[1, 1]], device=DEV))
    assert (cache[0, 0, -1, -9:] == 7).all() and (cache[0, 0, 5] == 3).all() and (cache[0, 0, 6] == 0).all()


def test_beam_reorder_in_a_graph_and_for_autograd():
    cache, parents = torch.randn(8, 2, 30, 16, device=DEV), torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    na.beam_reorder([cache], parents)
    with torch.cuda.graph(graph):
        na.beam_reorder([cache], parents)
    for i in range(3):
        parents.copy_(parents_of(2, 4, i))
        want = plain_reorder(cache, parents)
        graph.replay()
        assert torch.equal(cache, want)
    # autograd knows that the cache is another one now
    version = cache._version
    w = torch.randn(16, device=DEV, requires_grad=True)
    y = (cache * w).sum()
    na.beam_reorder(cache, parents)
    assert cache._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- recorded calls -------------------------------------------------------------------------------------------------
def recorded(which):
    def reordered(cache, parents, lengths):
        mine = [cache.clone(), cache * 2]
        na.beam_reorder(mine, parents, lengths)
        return mine
    prefix = lambda s: (rand(4, 4, 9, 32, seed=s), rand(2, 2, 40, 32, seed=s + 1), rand(2, 2, 40, 32, seed=s + 2))
    own = lambda s: (rand(4, 2, 12, 32, seed=s + 3), rand(4, 2, 12, 32, seed=s + 4))
    lengths = lambda s: (torch.tensor([12, 3 + s, 0, 9], device=DEV), torch.tensor([40 - s, 7], device=DEV))
    return {
        "prefix": (lambda q, pk, pv: na.prefix_attention(q, pk, pv, scale=0.25), prefix),
        "prefix_bf16": (lambda q, pk, pv, k, v: na.prefix_attention(q, pk, pv, k, v, 0.25, True), lambda s: tuple(t.to(BF16) for t in prefix(s) + own(s))),
        "prefix_lengths": (lambda q, pk, pv, k, v, n, p: na.prefix_attention(q, pk, pv, k, v, 0.25, True, n, p), lambda s: prefix(s) + own(s) + lengths(s)),
        "select": (lambda x, c, f: na.beam_select(x, c, 5, f, 2), lambda s: (*beams(2, 3, 50, F32, s), parents_of(2, 3, s) == 0)),
        "reorder": (reordered, lambda s: (rand(6, 2, 9, 16, seed=s), parents_of(2, 3, s), torch.arange(6, device=DEV) + s)),
    }[which]


def results(f, args, grad):
    args = [t.detach().requires_grad_(grad and t.is_floating_point()) for t in args]
    out = f(*args)
    out = list(out) if isinstance(out, (tuple, list)) else [out]
    if not grad:
        return out
    return [t.detach() for t in out] + list(torch.autograd.grad(out, [t for t in args if t.requires_grad], [torch.cos(t.detach()) for t in out]))


CALLS = [(w, g) for w in ("prefix", "prefix_bf16", "prefix_lengths") for g in (False, True)] + [("select", False), ("reorder", False)]


@pytest.mark.parametrize("which,grad", CALLS)
def test_a_traced_call_runs_again(which, grad):
    f, make = recorded(which)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, make(0), check_trace=False)
        for seed in (1, 2, 3):
            got, want = results(traced, make(seed), grad), results(f, make(seed), grad)
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which,grad", CALLS)
def test_a_call_recorded_by_a_dispatch_mode_runs_again(which, grad):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, make = recorded(which)
    with torch.set_grad_enabled(grad):
        graph = make_fx(lambda *args: results(f, args, grad))(*make(0))
        got, want = graph(*make(1)), results(f, make(1), grad)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


# ---- beside and behind other work ---------------------------------------------------------------------------------------
TOKENS = [(1, 64, 8, 2, 3000, 1, 200, 128), (16, 4, 16, 4, 1000, 1, 100, 64), (2, 6, 4, 2, 900, 5, 100, 128), (1, 2, 16, 2, 260, 5, 400, 64)]


@pytest.mark.parametrize("shape", TOKENS, ids=str)
def test_tokens_right_behind_what_writes_their_inputs(shape):
    """Kernels start under the ones before them: every input, the lengths too, is written just before the call that reads it."""
    S, A, N, Nk, P, Tq, Tk, C = shape
    sources = [operands(*shape, BF16, seed=10 * i)[:5] for i in range(3)]
    own = [torch.randint(Tq, Tk + 1, (S * A,), generator=torch.Generator().manual_seed(i)).int().to(DEV) for i in range(3)]
    prompts = [torch.randint(1, P + 1, (S,), generator=torch.Generator().manual_seed(i)).int().to(DEV) for i in range(3)]
    at = [t.clone() for t in sources[0]]
    lengths, prefix_lengths = own[0].clone(), prompts[0].clone()

    def call(i):
        for t, source in zip(at, sources[i]):
            t.copy_(source)
        prefix_lengths.copy_(prompts[i])
        lengths.copy_(own[i])
        return na.prefix_attention(*at, C ** -0.5, True, lengths, prefix_lengths)
    want = []
    for i in range(3):
        want.append(call(i))
        torch.cuda.synchronize()
    got = [call(i % 3) for i in range(30)]
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 3]), i
    na.check_kernels(DEV)


def test_calls_on_two_streams_at_once():
    shapes = TOKENS[:2]
    inputs = [operands(*shape, BF16, seed=i)[:5] for i, shape in enumerate(shapes)]
    logits = [beams(8, 4, 30011, BF16, i) for i in range(2)]
    caches = [torch.randn(8, 4, 500, 64, device=DEV) for _ in range(2)]
    parents = [parents_of(2, 4, i) for i in range(2)]

    def work(i):
        o = na.prefix_attention(*inputs[i], 0.125, True)
        moved = caches[i].clone()
        na.beam_reorder([moved], parents[i])
        return (o, *na.beam_select(*logits[i], 8), moved)
    want = [work(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    na.check_kernels(DEV)


def test_choices_and_caches_right_behind_what_writes_them():
    sources = [beams(6, 4, 40003, F16, i) for i in range(3)]
    logits, scores = (t.clone() for t in sources[0])
    cache, state = torch.zeros(24, 2, 300, 64, device=DEV), torch.randn(24, 2, 300, 64, device=DEV)

    def call(i):
        logits.copy_(sources[i][0])
        scores.copy_(sources[i][1])
        cache.copy_(state)
        found = na.beam_select(logits, scores)
        na.beam_reorder(cache, found[1])
        return (*found, cache.clone())
    want = []
    for i in range(3):
        want.append(call(i))
        torch.cuda.synchronize()
        assert torch.equal(want[-1][3], plain_reorder(state, want[-1][1]))
    for i, out in enumerate([call(i % 3) for i in range(30)]):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 3])), i


# ---- refusals -------------------------------------------------------------------------------------------------------
def test_prefix_attention_refuses():
    q, pk = torch.zeros(4, 4, 3, 32, device=DEV, dtype=BF16), torch.zeros(2, 2, 9, 32, device=DEV, dtype=BF16)
    k = torch.zeros(4, 2, 5, 32, device=DEV, dtype=BF16)
    n, p = torch.zeros(4, device=DEV, dtype=torch.int32), torch.zeros(2, device=DEV, dtype=torch.int32)
    na.prefix_attention(q, pk, pk, k, k, key_lengths=n, prefix_lengths=p)
    for args, kw in [((q, pk, pk[:, :, :5], k, k), {}), ((q, pk[:, :, :, :16], pk[:, :, :, :16], k, k), {}), ((q[:3], pk, pk, k[:3], k[:3]), {}),
                     ((q[:, :3], pk, pk, k, k), {}), ((q, pk, pk, k, None), {}), ((q, pk, pk, None, k), {}), ((q, pk, pk, k[:2], k[:2]), {}),
                     ((q, pk, pk, k[:, :1], k[:, :1]), {}), ((q, pk, pk, k.float(), k), {}), ((q, pk.float(), pk, k, k), {}), ((q, pk, pk, k.cpu(), k), {}),
                     ((q, pk[0], pk[0], k, k), {}), ((q, pk[:0], pk[:0], k, k), {}), ((q, pk, pk, k, k), dict(key_lengths=p)),
                     ((q, pk, pk, k, k), dict(prefix_lengths=n)), ((q, pk, pk), dict(key_lengths=n)), ((q, pk, pk, k, k), dict(key_lengths=n.float())),
                     ((q, pk, pk, k, k), dict(prefix_lengths=p.cpu())), ((q, pk, pk, k, k), dict(scale=0.0)), ((q, pk, pk, k, k), dict(scale=-1.0)),
                     ((q, pk, pk, k, k), dict(scale=math.nan)), ((q, torch._neg_view(pk), pk, k, k), {}),
                     ((q, pk, pk, k, k), dict(prefix_lengths=torch._neg_view(p)))]:
        with pytest.raises(ValueError):
            na.prefix_attention(*args, **kw)
    wide = torch.zeros(2, 2, 3, 260, device=DEV)
    with pytest.raises(ValueError):
        na.prefix_attention(wide, wide, wide)
    with pytest.raises(ValueError):
        na.prefix_attention_with_lse(q.float(), pk.float(), pk.float(), path="tensor")
    with pytest.raises(KeyError):
        na.prefix_attention_with_lse(q, pk, pk, path="other")


def test_prefix_attention_refuses_what_saved_tensor_hooks_hand_back():
    *x, d_o = operands(2, 2, 4, 2, 40, 9, 12, 32, BF16)
    n = torch.full((4,), 12, device=DEV, dtype=torch.int32)
    for change in (lambda t: t[:1] if t.dim() == 1 else t, lambda t: t.float() if t.dtype == BF16 and t.shape[0] == 2 else t,
                   lambda t: t[:, :, :5] if t.shape == (4, 4, 9, 32) else t, lambda t: t.double() if t.dim() == 3 else t):
        leaves = [t.detach().requires_grad_() for t in x]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            o = na.prefix_attention(*leaves, 0.2, True, n)
            with pytest.raises(ValueError):
                torch.autograd.grad(o, leaves, d_o)


def test_prefix_attention_is_not_differentiable_twice():
    x = [t.requires_grad_() for t in operands(1, 2, 2, 2, 20, 5, 5, 16, F32)[:5]]
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(na.prefix_attention(*x).sum(), x, create_graph=True)


def test_beam_select_refuses():
    logits, scores = beams(2, 3, 50, F32)
    ok = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    na.beam_select(logits, scores, 4, ok, 49)
    for args, kw in [((logits[0], scores), {}), ((logits, scores[:, :2]), {}), ((logits, scores.double()), {}), ((logits.double(), scores), {}),
                     ((logits, scores.cpu()), {}), ((logits, scores, 0), {}), ((logits, scores, -1), {}), ((logits, scores, 65), {}),
                     ((logits, scores), dict(end=50)), ((logits, scores), dict(end=-1)), ((logits, scores), dict(finished=ok.int())),
                     ((logits, scores), dict(finished=ok[:1])), ((logits, scores), dict(finished=ok.cpu())), ((logits[:, :, :0], scores), {}),
                     ((logits[:, :0], scores[:, :0], 1), {}), ((torch._neg_view(logits), scores), {}),
                     ((torch.zeros(1, 33, 5, device=DEV), torch.zeros(1, 33, device=DEV)), {}),
                     ((logits.clone().requires_grad_(), scores), {}), ((logits, scores.clone().requires_grad_()), {})]:
        with pytest.raises(ValueError):
            na.beam_select(*args, **kw)
    with torch.no_grad():
        na.beam_select(logits.clone().requires_grad_(), scores)


def test_beam_reorder_refuses():
    cache, parents = torch.zeros(6, 2, 9, 16, device=DEV), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    lengths = torch.zeros(6, dtype=torch.int32, device=DEV)
    for args in [(cache[:5], parents), (cache, parents.float()), (cache, parents[0]), (cache.cpu(), parents), (cache, parents.cpu()),
                 (cache[:1].expand(6, 2, 9, 16), parents), (cache[:, :, :1].expand(6, 2, 9, 16), parents),
                 (torch.zeros(24, device=DEV).as_strided((6, 1, 3, 4), (2, 12, 4, 1)), parents),       # entries that overlap
                 (cache.transpose(2, 3), parents), (cache[..., ::2], parents), (cache.flatten(1)[:, ::2], parents), (cache, parents, lengths[:5]),
                 (cache, parents, lengths.float()), (cache, parents, lengths.cpu()), (cache.flatten(2), parents, lengths),
                 (cache.clone().requires_grad_(), parents), (torch._neg_view(cache), parents), (cache, torch.zeros(1, 33, dtype=torch.int64, device=DEV)),
                 (torch.zeros(33, 2, device=DEV), torch.zeros(1, 33, dtype=torch.int64, device=DEV))]:
        with pytest.raises(ValueError):
            na.beam_reorder(*args)


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_search_over_shared_prompts(dtype):
    """Some steps of a search with all three operators: the caches that follow their beams, behind a prompt that is stored once, give
    each beam what attention gives for its whole history, stored by itself."""
    S, K, N, Nk, C, P, steps, V = 2, 3, 4, 2, 32, 50, 6, 40
    B = S * K
    pk, pv = rand(S, Nk, P, C, dtype=dtype), rand(S, Nk, P, C, dtype=dtype, seed=1)
    prompts = torch.tensor([P, 31], device=DEV)
    of_word = [rand(V, heads, C, dtype=dtype, seed=2 + i) for i, heads in enumerate((N, Nk, Nk))]         # q, k, v of each word
    out = rand(N * C, V, seed=9, scale=0.3)
    keys, values = (torch.zeros(B, Nk, steps, C, device=DEV, dtype=dtype) for _ in range(2))
    said = torch.zeros(B, steps, dtype=torch.int64, device=DEV)
    words = torch.zeros(S, K, dtype=torch.int64, device=DEV)
    scores = torch.tensor([0.0] + [-math.inf] * (K - 1), device=DEV).repeat(S, 1)
    for t in range(steps):
        said[:, t] = words.flatten()
        q, k, v = (w[words.flatten()] for w in of_word)
        keys[:, :, t], values[:, :, t] = k, v
        lengths = torch.full((B,), t + 1, device=DEV)
        o = na.prefix_attention(q.unsqueeze(2), pk, pv, keys, values, C ** -0.5, causal=True, key_lengths=lengths, prefix_lengths=prompts)
        # every beam's history, behind its own copy of the prompt
        for b in range(B):
            n = int(prompts[b // K])
            history = [torch.cat((p[b // K, :, :n], w[said[b, :t + 1]].transpose(0, 1)), 1).unsqueeze(0) for p, w in ((pk, of_word[1]), (pv, of_word[2]))]
            close(o[b:b + 1], na.attention(q[b:b + 1].unsqueeze(2), *history, C ** -0.5), dtype, 2, f"beam {b} step {t}")
        logits = (o.float().flatten(1) @ out).view(S, K, V)
        scores, parents, words = na.beam_select(logits, scores)
        na.beam_reorder([keys, values], parents, lengths)
        na.beam_reorder(said, parents)
    na.check_kernels(DEV)
