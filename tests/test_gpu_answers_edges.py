"""prefix_attention, beam_select and beam_reorder where one half, one cache or one candidate is quite unlike the others, and calls that
something looks into."""
import contextlib
import math

import pytest
import torch
import torch.overrides
import torch.utils._python_dispatch

import e_natten_b200 as na
from test_gpu_answers import beams, bits, check, operands, parents_of, plain_reorder
from test_gpu_block import BF16, DEV, F16, rand

pytestmark = pytest.mark.gpu


# ---- attention over a prefix: halves whose values differ in size --------------------------------------------------
def gradients_and_bounds(q, pk, pv, k, v, d_o, scale):
    """The gradients of q, pk, pv, k, v in 64 bits, all keys seen, and how far the kernels' may be off, element by element.

    u, half a step of the operands' type, for each rounding: of the weights in the forward's product and of o, both of which reach dS through
    delta = dO . o; of the weights in dV's product; of each result, with half a step of fp16's smallest numbers.  32 bits hold all else:
    products of up to 128 channels within 2^-17 of their terms' sizes, weights within 2^-16 of themselves (exponents of up to 32 in
    32 bits, and lse), sums of up to 512 terms within 2^-15 of the terms' sizes.  dS goes into its products as two numbers of 16 bits, u^2 of
    itself, in fp16 on a grid of 2^-37 of the largest |dO| |V| that it may have."""
    u, tiny = torch.finfo(q.dtype).eps / 2, 2.0 ** -25 if q.dtype == F16 else 0.0
    S, A, G = len(pk), len(q) // len(pk), q.shape[1] // pk.shape[1]
    P = pk.shape[2]
    q, pk, pv, k, v, g = (t.double() for t in (q, pk, pv, k, v, d_o))
    kk = torch.cat((pk.repeat_interleave(A, 0), k), 2).repeat_interleave(G, 1)
    vv = torch.cat((pv.repeat_interleave(A, 0), v), 2).repeat_interleave(G, 1)
    p = torch.softmax(q @ kk.mT * scale, -1)
    dp = g @ vv.mT
    o, delta = p @ vv, (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    of_o = u * (p @ vv.abs()) + u * o.abs() + tiny
    of_delta = (g.abs() * of_o).sum(-1, keepdim=True) + 2.0 ** -17 * (g * o).abs().sum(-1, keepdim=True)
    grid = 2.0 ** -37 * (g.norm(dim=-1).amax() * vv.norm(dim=-1).amax()) if tiny else 0.0
    of_ds = (p * (of_delta + 2.0 ** -17 * (g.abs() @ vv.abs().mT)) + (2.0 ** -16 + 2 * u * u) * p * (dp - delta).abs() + grid) * scale
    of_p = u * p + (2.0 ** -31 if tiny else 0.0)

    def keys(t):                                         # (B, heads, keys, C) -> prefix's, own
        t = t.unflatten(1, (-1, G)).sum(2)
        return t[:, :, :P].unflatten(0, (S, A)).sum(1), t[:, :, P:]
    sums = 2.0 ** -15
    dq, dq_off = ds @ kk, of_ds @ kk.abs() + sums * (ds.abs() @ kk.abs())
    dk, dk_off = keys(ds.mT @ q), keys(of_ds.mT @ q.abs() + sums * (ds.abs().mT @ q.abs()))
    dv, dv_off = keys(p.mT @ g), keys(of_p.mT @ g.abs() + sums * (p.mT @ g.abs()))
    want = (dq, dk[0], dv[0], dk[1], dv[1])
    return want, [off + u * t.abs() + tiny for off, t in zip((dq_off, dk_off[0], dv_off[0], dk_off[1], dv_off[1]), want)]


@pytest.mark.parametrize("Tq", [1, 40])
@pytest.mark.parametrize("of_prefix,of_own,of_do", [(2.0 ** -12, 1.0, 1.0), (1.0, 2.0 ** -12, 1.0), (0.0, 1.0, 1.0), (1.0, 0.0, 1.0), (0.0, 1.0, 2.0 ** -12),
                                                    (1.0, 0.0, 2.0 ** -12), (2.0 ** 12, 1.0, 2.0 ** -8), (1.0, 2.0 ** 12, 2.0 ** -8), (2.0 ** -12, 2.0 ** 8, 2.0 ** -6),
                                                    (0.0, 0.0, 1.0)])
@pytest.mark.parametrize("scale", [0.125, 0.5], ids=["even", "peaked"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_prefix_attention_gradients_of_halves_of_any_size(dtype, scale, of_prefix, of_own, of_do, Tq):
    """Values of the prompt far above, far below, and beside the answers' own, none of them (0) too: delta = dO . o holds both.  Values of a
    half, and dO, point the same way, so that dP and delta are as large as their norms allow; queries are large and keys small, so that dS
    of small values still count."""
    S, A, N, Nk, P, Tk, C = 2, 3, 4, 2, 70, 40, 64
    q, pk, pv, k, v, d_o = operands(S, A, N, Nk, P, Tq, Tk, C, dtype)
    way = rand(2, 1, Nk, 1, C, seed=11)
    large = 2.0 ** 8 if of_do < 1.0 and of_prefix * of_own == 0 else 1.0
    q, pk, k = (q.float() * large).to(dtype), (pk.float() / large).to(dtype), (k.float() / large).to(dtype)
    pv, v = ((way[i] + 0.1 * t.float()).mul(by).to(dtype) for i, t, by in ((0, pv, of_prefix), (1, v, of_own)))
    d_o = (way.sum(0).repeat_interleave(N // Nk, 1) + 0.1 * d_o.float()).mul(of_do).to(dtype)
    leaves = [t.requires_grad_() for t in (q, pk, pv, k, v)]
    got = torch.autograd.grad(na.prefix_attention(*leaves, scale), leaves, d_o)
    na.check_kernels(DEV)
    want, off = gradients_and_bounds(*(t.detach() for t in leaves), d_o, scale)
    for name, a, ref, most in zip(("dq", "dpk", "dpv", "dk", "dv"), got, want, off):
        assert torch.isfinite(a).all(), name
        assert ref.abs().max() < 60000, "the test's own values fit"
        far = ((a.double() - ref).abs() / most.clamp_min(1e-300)).max()
        assert far <= 1, f"{name}: {far:.3g} times as far off as roundings account for"


# ---- attention over a prefix: head dims above 128, whose key half has instances of its own --------------------------
@pytest.mark.parametrize("dtype,C", [(torch.float32, 130), (BF16, 136), (F16, 256)])
@pytest.mark.parametrize("S,A,N,Nk,P,Tq,Tk", [(2, 3, 4, 2, 66, 20, 21), (1, 8, 4, 1, 40, 100, 100), (2, 2, 2, 2, 130, 40, 0)])       # in the second the prompt's are in parts
def test_prefix_attention_gradients_of_some_keys_at_wide_heads(S, A, N, Nk, P, Tq, Tk, dtype, C):
    """Both halves' keys, and either half's alone: two problems of a launch, the first, the second."""
    *x, d_o = operands(S, A, N, Nk, P, Tq, Tk, C, dtype)
    _, want = check(*x, d_o, C ** -0.5, True)
    names = ("q", "pk", "pv", "k", "v")[:5 if Tk else 3]
    for some in (("pk", "pv"), ("k", "v"), ("q", "v"), ("q", "pk"), ("pv", "k")):
        some = [n for n in some if n in names]
        if not some:
            continue
        leaves = {n: t.detach().requires_grad_(n in some) for n, t in zip(names, x)}
        o = na.prefix_attention(*leaves.values(), *((None, None) if not Tk else ()), C ** -0.5, True)
        got = torch.autograd.grad(o, [leaves[n] for n in some], d_o)
        for n, g in zip(some, got):
            assert torch.equal(g, want[names.index(n)]), (some, n)
    na.check_kernels(DEV)


# ---- beam search: calls that something looks into --------------------------------------------------------------------
class Through(torch.utils._python_dispatch.TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def a_cache(seed=0, B=2, K=4):
    return rand(B * K, 2, 30, 16, seed=seed), parents_of(B, K, seed)


def test_beam_reorder_under_a_dispatch_mode_tells_autograd():
    """What was recorded before is not differentiated with the values of after."""
    cache, parents = a_cache()
    want, version = plain_reorder(cache, parents), cache._version
    w = rand(16).requires_grad_()
    y = (cache * w).sum()
    with Through():
        na.beam_reorder(cache, parents)
    assert torch.equal(cache, want) and cache._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        mine = cache.clone()
    with Through():
        na.beam_reorder(mine, parents)                   # (no version to count)
    assert torch.equal(mine, plain_reorder(cache, parents))


@pytest.mark.parametrize("mode", [lambda: torch.device("cuda"), torch.overrides.TorchFunctionMode])
def test_beam_reorder_under_a_function_mode_is_in_place(mode):
    """No second copy of a cache, as without one."""
    cache = torch.randn(8, 4, 512, 256, device=DEV)
    parents = parents_of(2, 4, 5)
    want, version = plain_reorder(cache, parents), cache._version
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with mode():
        na.beam_reorder(cache, parents)
    assert torch.cuda.max_memory_allocated() - before < cache.nbytes // 4
    assert torch.equal(cache, want) and cache._version > version


def test_beam_operators_refuse_tensors_with_tangents():
    cache, parents = a_cache()
    logits, scores = beams(2, 4, 50, torch.float32)
    was = cache.clone()
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: na.beam_reorder(dual(cache), parents), lambda: na.beam_reorder([cache, dual(cache)], parents),
                     lambda: na.beam_select(dual(logits), scores), lambda: na.beam_select(logits, dual(scores))):
            with pytest.raises(ValueError, match="no gradient"):
                call()
    assert torch.equal(cache, was)


@pytest.mark.parametrize("mode", [Through, contextlib.nullcontext])
def test_beam_reorder_checks_every_cache_before_it_moves_one(mode):
    good, parents = a_cache()
    was = good.clone()
    for bad in (good[:7].clone(), good[:1].clone().expand(8, 2, 30, 16), good.clone().transpose(2, 3), good.cpu(), torch._neg_view(good.clone())):
        with mode(), pytest.raises(ValueError):
            na.beam_reorder([good, bad], parents)
    with mode(), pytest.raises(ValueError):
        na.beam_reorder([good, good.flatten(2)], parents, torch.zeros(8, dtype=torch.int32, device=DEV))
    with mode(), pytest.raises(ValueError):
        na.beam_reorder([good, good.clone().requires_grad_()], parents)
    assert torch.equal(good, was)


def test_beam_reorder_of_caches_of_unlike_rows():
    """Rows of 16 bytes' multiples, of 4's and of single bytes in one list, each in pieces of its own; more of one kind than a launch takes."""
    B, K, T = 2, 4, 70
    parents = parents_of(B, K, 9)
    lengths = (torch.arange(B * K, device=DEV) * 11).int()
    like = lambda: [bits(B * K, 2, T, 64, dtype=torch.int16, seed=1), bits(B * K, 1, T, 13, dtype=torch.int32, seed=2), bits(B * K, 3, T, 5, seed=3),
                    bits(B * K, 1, T, 1, dtype=torch.bool, seed=4), bits(B * K, T, 2, 8, dtype=torch.int64, seed=5).transpose(1, 2),
                    *(bits(B * K, 1, T, 3 + i % 2, dtype=torch.int32, seed=6 + i) for i in range(150))]
    for n in (None, lengths):
        caches = like()
        want = [plain_reorder(c, parents, n) for c in caches]
        na.beam_reorder(caches, parents, n)
        assert all(torch.equal(a, b) for a, b in zip(caches, want))


# ---- beam search: how far off a worth may be ---------------------------------------------------------------------------
def most_off(logits):
    """How far the logarithm of each row's sum may be off.  An exponent, a difference of 32 bits times 1 / ln 2 in 32 bits, is off by (2^-24 +
    2^-24 + 2^-26) of itself: that, by the words' weights; an exponential by 2^-22 of itself, and a sum is multiplied by one for each chunk of a
    block, up to 16, and once more; 52 roundings of 2^-24 (8 sums in a chunk, 16 chunks, their 15 factors, 13 to join a block's threads).  Blocks
    are joined in 64 bits."""
    x = logits.double()
    distance = (torch.softmax(x, -1) * (x.amax(-1, keepdim=True) - x)).sum(-1)
    return 2.25 * 2.0 ** -24 * distance + 17 * 2.0 ** -22 + 52 * 2.0 ** -24


def rows_of_sums(V):
    """Rows whose sums are hard: a peak before equal words far below it, words that climb from chunk to chunk, equal words."""
    tails = [0.1, 1.7, 5.3, 8.9, 10.2, 11.37, 12.7, 13.1, 14.9, 15.9, 17.3, 20.1]
    x = torch.zeros(len(tails) + 4, V, device=DEV)
    for row, tail in zip(x, tails):
        row[1:] = -tail
        row[0] = 0.37
    line = torch.arange(V, device=DEV, dtype=torch.float64) / V
    x[-4], x[-3], x[-2], x[-1] = 1e-3 * line, 7.3 * line, 30 * line, -0.123
    return x


@pytest.mark.parametrize("V", [1000, 50257, 1 << 18, 1 << 22])
def test_beam_select_worths_of_uneven_rows(V):
    x = rows_of_sums(V)
    for dtype in (torch.float32, BF16):
        logits = x.to(dtype)
        want = logits.double().amax(-1) - logits.double().logsumexp(-1)
        got = na.beam_select(logits[:, None], torch.zeros(len(x), 1, device=DEV))[0][:, 0]
        off = (got.double() - want).abs()
        most = most_off(logits)
        assert most.max() < 2.0 ** -16.5                 # what the documents say, and the score's own rounding
        assert (off <= most + 2.0 ** -24 * want.abs()).all()


def test_beam_select_orders_worths_that_are_far_enough_apart():
    """Beams of one peak each before tails of their own, in the order that 64 bits give where worths are 2^-15 apart."""
    V, apart = 1 << 18, 2.0 ** -15
    x = rows_of_sums(V)
    ends = x.double().amax(-1) - x.double().logsumexp(-1)
    order = torch.randperm(len(x), generator=torch.Generator().manual_seed(3)).to(DEV)
    worths = -1.0 - apart * 1.001 * order.double()       # of each beam's best
    scores = (worths - ends).float()
    have = scores.double() + ends                        # (scores are rounded to 32 bits)
    best = torch.argsort(have, descending=True)
    assert (have[best][:-1] - have[best][1:] > apart * 0.9).all()
    parents = na.beam_select(x[None, :-4], scores[None, :-4], 1)[1]
    kept = best[best < len(x) - 4]
    assert parents[0, 0] == kept[0]
    for _ in range(len(kept) - 1):                       # the best beam of those left, one after the other
        scores[kept[0]] = -math.inf
        kept = kept[1:]
        assert na.beam_select(x[None, :-4], scores[None, :-4], 1)[1][0, 0] == kept[0]


@pytest.mark.parametrize("mode", [contextlib.nullcontext, Through])
def test_beam_reorder_of_what_says_how(mode):
    """Parents, or lengths, that are themselves among the caches: all move by what they were."""
    B, K, T = 4, 8, 4000
    for seed in range(5):
        parents, cache = parents_of(B, K, seed), bits(B * K, 1, T, 9, dtype=torch.int32, seed=seed)
        lengths = torch.randint(0, T + 1, (B * K,), generator=torch.Generator().manual_seed(seed)).to(DEV)
        said = parents.view(-1)
        want = [plain_reorder(t, parents.clone()) for t in (said, cache)]
        with mode():
            na.beam_reorder([said, cache], parents)
        assert torch.equal(said, want[0]) and torch.equal(cache, want[1])
        parents = parents_of(B, K, seed + 10)
        held = lengths.view(-1, 1, 1, 1)
        want = [plain_reorder(t, parents, lengths.clone()) for t in (held, cache)]
        with mode():
            na.beam_reorder([held, cache], parents, lengths)
        assert torch.equal(held, want[0]) and torch.equal(cache, want[1])
