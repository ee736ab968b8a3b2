"""group_norm, rotary and attention against plain implementations in 64 bits, at the sizes and masks where they can go
wrong, and their refusals.

Tolerances, from what is rounded (u: the unit roundoff, 2^-8 bf16, 2^-11 fp16):
 * a 16-bit result is rounded once, by up to u of each element.  Attention also rounds P, and the backward P or dS, to 16 bits for
   their products, and forms delta from the rounded o.  A rounding's root mean square is at most u / sqrt(3): two of them
   make less than u in the norm (o), three, of which one meets a difference, less than 1.5 u (the gradients), and no element is
   off by more than 8 times that of its own size or the tensor's rms, whichever is larger.
 * A gradient whose terms p dp k cancel (nearly all weight on one key: dp - delta is far smaller than dp) is off by the roundings of
   the terms, not of what is left of them: it is measured against the root of their summed squares where that is larger.
 * 32-bit results: 2^-24 for each step of sums that are taken over threads and tiles (a few hundred terms one after another at
   most, errors of either sign) and exponentials whose argument of up to 2^5 is off by 2^-24 of itself: 1e-5 for gradients.
"""
import ctypes
import math

import pytest
import torch

import e_natten_b200 as na
from e_natten_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 6.7e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def close(got, want, dtype, units, what, terms=0.0):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} is not {tuple(want.shape)}"
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if want.numel() == 0:
        return
    bound, rms = units * U[dtype], want.square().mean().sqrt().clamp_min(terms)
    if rms == 0:
        assert (got == 0).all(), f"{what}: not zero"
        return
    err = (got - want).abs()
    norm = err.square().mean().sqrt() / rms
    worst = (err / want.abs().clamp_min(rms)).max()
    assert norm <= bound and worst <= 8 * bound, f"{what}: {norm:.2e} in the norm, {worst:.2e} at worst, of {bound:.2e}"


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale + shift).to(dtype).to(DEV)


# ---- attention ----------------------------------------------------------------------------------------------
def plain_attention(q, k, v, d_o, scale, causal, lengths):
    """(o, lse, dq, dk, dv) in 64 bits, head by head over the keys that a row sees, and for each batch entry the rms of the
    root of dq's and of dk's terms' summed squares."""
    B, N, Tq, C = q.shape
    Nk, Tk = k.shape[1:3]
    q, k, v, g = (t.double() for t in (q, k, v, d_o))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lse = torch.full((B, N, Tq), -math.inf, dtype=torch.float64, device=q.device)
    squares_q, squares_k = q.new_zeros(B), q.new_zeros(B)
    for b in range(B):
        L = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        row = torch.arange(Tq, device=q.device)
        seen = (L - Tq + 1 + row).clamp(0, L) if causal else torch.full_like(row, L)
        mask = torch.arange(L, device=q.device) < seen[:, None]
        ok = seen > 0
        if not ok.any():
            continue
        for n in range(N):
            m = n // (N // Nk)
            kk, vv = k[b, m, :L], v[b, m, :L]
            s = (q[b, n, ok] @ kk.T * scale).masked_fill(~mask[ok], -math.inf)
            lse[b, n, ok] = s.logsumexp(-1)
            p = (s - s.logsumexp(-1, keepdim=True)).exp()
            o[b, n, ok] = p @ vv
            dp = g[b, n, ok] @ vv.T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            dq[b, n, ok] = ds @ kk
            dk[b, m, :L] += ds.T @ q[b, n, ok]
            dv[b, m, :L] += p.T @ g[b, n, ok]
            terms = (p * dp * scale).square()
            squares_q[b] += (terms @ kk.square()).sum()
            squares_k[b] += (terms.T @ q[b, n, ok].square()).sum() * (Tk / L)
    return o, lse, dq, dk, dv, (squares_q / (N * Tq * C)).sqrt(), (squares_k / (Nk * Tk * C)).sqrt()


def check_attention(q, k, v, d_o, scale=None, causal=False, lengths=None, path="auto", what=""):
    dtype = q.dtype
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o, lse = na.attention_with_lse(q, k, v, scale, causal, lengths, path)
    grads = torch.autograd.grad(o, (q, k, v), d_o)
    na.check_kernels(DEV)
    want = plain_attention(q.detach(), k.detach(), v.detach(), d_o, 1.0 if scale is None else scale, causal, lengths)
    seen = want[1] > -math.inf
    for b in range(len(q)):
        close(o.detach()[b][seen[b]], want[0][b][seen[b]], dtype, 1, f"o {b} {what}")
    assert (o[~seen] == 0).all() and (grads[0][~seen] == 0).all()
    assert torch.equal(lse == -math.inf, ~seen), f"lse {what}: rows that see nothing"
    if seen.any():
        assert (lse.double() - want[1])[seen].abs().max() < 1e-4, f"lse {what}"        # fp32 of numbers up to about 2^4, of 16-bit operands exactly
    for b in range(len(q)):         # entries of different lengths have gradients of different sizes: each by itself, over its rows and keys
        L = k.shape[2] if lengths is None else min(max(int(lengths[b]), 0), k.shape[2])
        rows = seen[b]
        close(grads[0][b][rows], want[2][b][rows], dtype, 1.5, f"dq {b} {what}", want[5][b] * (rows.numel() / max(1, int(rows.sum()))) ** 0.5)
        close(grads[1][b, :, :L], want[3][b, :, :L], dtype, 1.5, f"dk {b} {what}", want[6][b])
        close(grads[2][b, :, :L], want[4][b, :, :L], dtype, 1.5, f"dv {b} {what}")
        assert (grads[1][b, :, L:] == 0).all() and (grads[2][b, :, L:] == 0).all()
    return o.detach(), grads


SHAPES = [  # B, N, Nk, Tq, Tk, C
    (1, 1, 1, 1, 1, 32), (1, 2, 2, 3, 5, 64), (2, 3, 3, 64, 64, 64), (2, 2, 2, 128, 128, 128), (1, 2, 2, 129, 127, 128),
    (2, 4, 2, 196, 196, 64), (1, 6, 2, 300, 77, 32), (1, 8, 1, 17, 260, 128), (2, 2, 1, 257, 513, 128), (3, 4, 4, 31, 700, 48),
    (1, 2, 2, 130, 140, 96), (1, 1, 1, 640, 384, 8), (1, 12, 4, 40, 129, 128),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_on_tensor_cores(shape, dtype, causal):
    B, N, Nk, Tq, Tk, C = shape
    q, k, v = rand(B, N, Tq, C, dtype=dtype), rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    check_attention(q, k, v, rand(B, N, Tq, C, dtype=dtype, seed=3), C ** -0.5, causal, path="tensor")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES + [(1, 2, 1, 70, 90, 200), (2, 2, 2, 33, 65, 7), (1, 1, 1, 65, 64, 130)], ids=str)
def test_attention_in_32_bits(shape, causal):
    B, N, Nk, Tq, Tk, C = shape
    q, k, v = rand(B, N, Tq, C), rand(B, Nk, Tk, C, seed=1), rand(B, Nk, Tk, C, seed=2)
    check_attention(q, k, v, rand(B, N, Tq, C, seed=3), C ** -0.5, causal)


@pytest.mark.parametrize("dtype,C", [(BF16, 7), (F16, 36), (BF16, 136)])
def test_attention_head_dims_without_tensor_cores(dtype, C):
    q, k, v = rand(1, 4, 75, C, dtype=dtype), rand(1, 2, 66, C, dtype=dtype, seed=1), rand(1, 2, 66, C, dtype=dtype, seed=2)
    check_attention(q, k, v, rand(1, 4, 75, C, dtype=dtype, seed=3), C ** -0.5, lengths=torch.tensor([50], device=DEV))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,Nk,Tq,Tk,C", [(4, 2, 70, 300, 64), (2, 2, 200, 256, 128), (8, 2, 5, 1000, 32), (3, 3, 140, 130, 128)])
def test_attention_lengths(N, Nk, Tq, Tk, C, dtype, causal):
    """Every length at which a tile can end, none among them; what lies beyond is not looked at, and gets no gradient."""
    lengths = torch.tensor([0, 1, 2, 63, 64, 127, 128, 129, Tk - 1, Tk, Tk + 9, -3], device=DEV)
    B = len(lengths)
    q, k, v = rand(B, N, Tq, C, dtype=dtype), rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    d_o = rand(B, N, Tq, C, dtype=dtype, seed=3)
    o, grads = check_attention(q, k, v, d_o, C ** -0.5, causal, lengths)
    beyond = torch.arange(Tk, device=DEV) >= lengths[:, None]
    poisoned_k, poisoned_v = (t.masked_fill(beyond[:, None, :, None], x) for t, x in ((k, math.inf), (v, math.nan)))
    for t in (q, poisoned_k, poisoned_v):
        t.requires_grad_()
    o2 = na.attention(q, poisoned_k, poisoned_v, C ** -0.5, causal, lengths.int())
    grads2 = torch.autograd.grad(o2, (q, poisoned_k, poisoned_v), d_o)
    assert torch.equal(o2, o)
    for name, x, y in zip(("dq", "dk", "dv"), grads2, grads):
        assert torch.equal(x, y), name
    for x in grads2[1:]:
        assert (x.masked_select(beyond[:, None, :, None]) == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,N,Nk,Tq,Tk,C", [(2, 8, 2, 1, 5000, 128), (1, 4, 4, 1, 9000, 64), (3, 2, 1, 2, 4111, 96), (1, 2, 2, 130, 4000, 32),
                                            (1, 32, 1, 1, 3000, 128), (2, 6, 3, 5, 2049, 64)])
def test_attention_of_few_queries_in_parts(B, N, Nk, Tq, Tk, C, dtype):
    """The forms of serving: the keys of a row are taken in parts, also where lengths leave some of them empty."""
    q, k, v = rand(B, N, Tq, C, dtype=dtype), rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    lengths = torch.tensor([Tk, 600, 0][:B], device=DEV, dtype=torch.int32)
    for use in (None, lengths):
        with torch.no_grad():
            o, lse = na.attention_with_lse(q, k, v, C ** -0.5, True, use)
        na.check_kernels(DEV)
        want = plain_attention(q, k, v, q, C ** -0.5, True, use)
        close(o, want[0], dtype, 1, "o")
        seen = want[1] > -math.inf
        assert torch.equal(lse == -math.inf, ~seen) and (lse.double() - want[1])[seen].abs().max() < 1e-4


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_of_few_keys_in_parts(dtype):
    q, k, v = rand(2, 8, 1500, 64, dtype=dtype), rand(2, 2, 100, 64, dtype=dtype, seed=1), rand(2, 2, 100, 64, dtype=dtype, seed=2)
    check_attention(q, k, v, rand(2, 8, 1500, 64, dtype=dtype, seed=3), 0.125, lengths=torch.tensor([100, 37], device=DEV))


@pytest.mark.parametrize("dtype,C", [(BF16, 64), (F16, 128), (BF16, 32)])
@pytest.mark.parametrize("B,N,Nk,Tq,Tk,lengths", [
    (10, 5, 5, 1024, 384, None),                                      # 150 tiles of keys: a second round for two of them
    (7, 4, 2, 700, 300, [300, 0, 129, 1, 128, 299, 0]),               # some tiles hold no key
    (3, 2, 1, 1100, 900, [0, 0, 0]),
    (3, 2, 2, 1030, 140, [0, 140, 0]),
])
def test_attention_shares_the_queries_out(B, N, Nk, Tq, Tk, lengths, dtype, C):
    """The key half, where its CTAs take equal stretches of all tiles' queries."""
    q, d_o = rand(B, N, Tq, C, dtype=dtype), rand(B, N, Tq, C, dtype=dtype, seed=3)
    k, v = rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    check_attention(q, k, v, d_o, C ** -0.5, lengths=None if lengths is None else torch.tensor(lengths, device=DEV))


@pytest.mark.parametrize("dtype,C", [(BF16, 64), (F16, 128), (F16, 32)])
@pytest.mark.parametrize("B,N,Nk,Tq,Tk,lengths", [
    (10, 5, 5, 384, 1024, None),                                      # 150 tiles of rows: a second round for two of them
    (3, 4, 2, 100, 3000, [3000, 0, 1537]),                            # few rows, many keys
    (2, 6, 1, 33, 2500, [0, 0]),
    (5, 15, 15, 300, 1100, [1100, 130, 0, 1, 1099]),
])
def test_attention_shares_the_keys_out(B, N, Nk, Tq, Tk, lengths, dtype, C):
    """The query half, where its CTAs take equal stretches of all tiles' keys."""
    q, d_o = rand(B, N, Tq, C, dtype=dtype), rand(B, N, Tq, C, dtype=dtype, seed=3)
    k, v = rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    check_attention(q, k, v, d_o, C ** -0.5, lengths=None if lengths is None else torch.tensor(lengths, device=DEV))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,C", [(BF16, 64), (F16, 128), (F16, 32)])
@pytest.mark.parametrize("B,N,Nk,Tq,Tk,lengths", [(1, 2, 2, 1500, 1500, None), (2, 4, 2, 1100, 1300, [1300, 700]), (1, 2, 1, 2100, 130, [130])])
def test_attention_gradients_in_parts_and_whole(B, N, Nk, Tq, Tk, lengths, dtype, C, causal):
    """With its workspace a backward cuts tiles into parts, without it does not: the same fp32 sums in another order (2e-5 of values of
    order one), rounded once to the type (a flip of its last bit)."""
    q, d_o = rand(B, N, Tq, C, dtype=dtype), rand(B, N, Tq, C, dtype=dtype, seed=3)
    k, v = rand(B, Nk, Tk, C, dtype=dtype, seed=1), rand(B, Nk, Tk, C, dtype=dtype, seed=2)
    lengths = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    o, lse = na.attention_with_lse(q, k, v, C ** -0.5, causal, lengths)
    a = _lib.AttentionArgs()
    a.struct_size = ctypes.sizeof(_lib.AttentionArgs)
    a.B, a.N, a.Nk, a.Tq, a.Tk, a.C, a.dtype, a.causal, a.scale = B, N, Nk, Tq, Tk, C, 1 if dtype == BF16 else 2, causal, C ** -0.5
    a.stream = torch.cuda.current_stream(DEV).cuda_stream
    delta = torch.empty_like(lse)
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o), ("d_o", d_o)):
        setattr(a, name, _lib.Heads(t.data_ptr(), 0, 0, 0))
    a.lse, a.delta = lse.data_ptr(), delta.data_ptr()
    if lengths is not None:
        a.key_lengths = lengths.data_ptr()
    results = []
    for whole in (False, True):
        out = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        for name, t in zip(("d_q", "d_k", "d_v"), out):
            setattr(a, name, _lib.Heads(t.data_ptr(), 0, 0, 0))
        room = _lib.lib.na2d_attention_workspace(ctypes.byref(a), 1)
        assert room > 0
        workspace = torch.empty(room, dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = (None, 0) if whole else (workspace.data_ptr(), room)
        _lib.check(_lib.lib.na2d_attention_backward(ctypes.byref(a)))
        na.check_kernels(DEV)
        results.append(out)
    for name, got, want in zip("qkv", *results):
        got, want = got.double(), want.double()
        assert torch.isfinite(want).all() and torch.isfinite(got).all(), name
        assert ((got - want).abs() <= 2 * U[dtype] * want.abs() + 2e-5).all(), name


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_on_grids_and_views(dtype):
    """(B, heads, H, W, C) views of a packed projection, a gradient with heads last, an image whose rows do not follow one another."""
    B, H, W, N, C = 2, 9, 13, 3, 64
    packed = rand(B, H, W, 3, N, C, dtype=dtype)
    q, k, v = packed.permute(3, 0, 4, 1, 2, 5).unbind(0)
    d_o = rand(B, H, W, N, C, dtype=dtype, seed=3).permute(0, 3, 1, 2, 4)
    crop = rand(B, N, H + 2, W + 3, C, dtype=dtype, seed=4)[:, :, 1:-1, 2:-1]
    for a, b, c in ((q, k, v), (crop, k, crop)):
        a, b, c = (t.detach().requires_grad_() for t in (a, b, c))
        o, lse = na.attention_with_lse(a, b, c, 0.125)
        assert o.shape == (B, N, H, W, C) and lse.shape == (B, N, H, W)
        grads = torch.autograd.grad(o, (a, b, c), d_o)
        want = plain_attention(*(t.detach().flatten(2, 3) for t in (a, b, c)), d_o.flatten(2, 3), 0.125, False, None)
        close(o.detach().flatten(2, 3), want[0], dtype, 1, "o")
        for name, got, ref in zip(("dq", "dk", "dv"), grads, want[2:]):
            close(got.flatten(2, 3), ref, dtype, 1.5, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_large_logits(dtype):
    """Unscaled logits: nearly all weight on one key, maxima that grow along the row."""
    q, k, v = rand(1, 2, 200, 64, dtype=dtype, scale=2.0), rand(1, 2, 400, 64, dtype=dtype, seed=1), rand(1, 2, 400, 64, dtype=dtype, seed=2)
    k = (k * torch.linspace(0.1, 3, 400, device=DEV)[:, None]).to(dtype)
    with torch.no_grad():
        o, lse = na.attention_with_lse(q, k, v)
    want = plain_attention(q, k, v, q, 1.0, False, None)
    # exponents' arguments reach 2^7: 2^-24 of that in each weight, in 32 bits
    close(o, want[0], dtype, 1 if dtype != F32 else 4, "o")
    assert ((lse.double() - want[1]).abs() <= 2e-6 * want[1].abs() + 1e-4).all()


def test_attention_infinite_logits_and_nan():
    q, k, v = (rand(1, 1, 130, 64, dtype=BF16, seed=i) for i in range(3))
    q[0, 0, 5] = math.nan
    k[0, 0, 7] = -math.inf
    with torch.no_grad():
        o = na.attention(q, k, v, 0.125)
    bad = torch.isnan(o).all(-1)[0, 0]
    s = (q[0, 0].double() @ k[0, 0].double().T) * 0.125
    assert torch.equal(bad, torch.isnan(torch.softmax(s, -1)).any(-1))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,N,Tq,Tk", [(0, 2, 4, 4), (2, 0, 4, 4), (2, 2, 0, 4), (2, 2, 4, 0)])
def test_attention_of_nothing(B, N, Tq, Tk, dtype):
    q, k, v = (torch.randn(B, N or n, t, 32, device=DEV, dtype=dtype)[:, :N or n].requires_grad_() for n, t in ((N, Tq), (1, Tk), (1, Tk)))
    if N == 0:
        q = torch.zeros(B, 0, Tq, 32, device=DEV, dtype=dtype, requires_grad=True)
    o, lse = na.attention_with_lse(q, k, v)
    assert o.shape == q.shape and (o == 0).all() and (lse == -math.inf).all()
    for t, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
        assert g.shape == t.shape and (g == 0).all()


def test_attention_is_the_same_every_time_and_on_any_stream():
    q, k, v = rand(2, 8, 500, 64, dtype=BF16), rand(2, 2, 900, 64, dtype=BF16, seed=1), rand(2, 2, 900, 64, dtype=BF16, seed=2)
    d_o = rand(2, 8, 500, 64, dtype=BF16, seed=3)

    def step():
        a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
        o = na.attention(a, b, c, 0.125, True)
        return (o.detach(), *torch.autograd.grad(o, (a, b, c), d_o))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, second):
        assert torch.equal(x, y)


def test_attention_needs_only_some_gradients():
    q, k, v = rand(1, 2, 140, 64, dtype=BF16), rand(1, 2, 150, 64, dtype=BF16, seed=1), rand(1, 2, 150, 64, dtype=BF16, seed=2)
    d_o = rand(1, 2, 140, 64, dtype=BF16, seed=3)
    whole = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(na.attention(*whole, 0.125), whole, d_o)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(na.attention(*some, 0.125), some[i], d_o)
        assert torch.equal(got, want[i])


def differences(f, t, g, entries, h):
    """Central differences of sum(f() * g) by entries of t."""
    found = []
    flat = t.view(-1)
    for i in entries:
        old = flat[i].item()
        flat[i] = old + h
        up = (f().double() * g.double()).sum()
        flat[i] = old - h
        down = (f().double() * g.double()).sum()
        flat[i] = old
        found.append(((up - down) / (2 * h)).item())
    return torch.tensor(found, dtype=torch.float64)


def test_attention_gradient_against_differences():
    q, k, v = rand(1, 4, 20, 16), rand(1, 2, 70, 16, seed=1), rand(1, 2, 70, 16, seed=2)
    d_o, lengths = rand(1, 4, 20, 16, seed=3), torch.tensor([66], device=DEV)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(na.attention(*leaves, 0.25, True, lengths), leaves, d_o)
    with torch.no_grad():
        for t, g in zip((q, k, v), grads):
            entries = list(range(3, t.numel(), t.numel() // 12))
            # truncation h^2, rounding of the sum (about 1e-6) over 2 h
            got = differences(lambda: na.attention(q, k, v, 0.25, True, lengths), t, d_o, entries, 1e-2)
            assert (got - g.view(-1)[entries].double().cpu()).abs().max() < 2e-3


# ---- group normalisation ---------------------------------------------------------------------------------------------
def plain_norm(x, groups, w, b, eps, silu, d_y):
    x64 = x.double().requires_grad_()
    params = [None if p is None else p.double().requires_grad_() for p in (w, b)]
    C = x.shape[-1]
    flat = x64.reshape(x.shape[0], -1, groups, C // groups)
    mean, var = flat.mean((1, 3), keepdim=True), flat.var((1, 3), correction=0, keepdim=True)
    z = ((flat - mean) / (var + eps).sqrt()).reshape(x.shape)
    if params[0] is not None:
        z = z * params[0]
    if params[1] is not None:
        z = z + params[1]
    y = z * torch.sigmoid(z) if silu else z
    leaves = [x64] + [p for p in params if p is not None]
    return y.detach(), torch.autograd.grad(y, leaves, d_y.double())


def check_norm(x, groups, w, b, d_y, activation="silu", eps=1e-5, units=1.0, param_units=1.0):
    leaves = [x.detach().requires_grad_()] + [p.detach().requires_grad_() for p in (w, b) if p is not None]
    args = iter(leaves[1:])
    y = na.group_norm(leaves[0], groups, next(args) if w is not None else None, next(args) if b is not None else None, eps, activation)
    grads = torch.autograd.grad(y, leaves, d_y)
    want, want_grads = plain_norm(x, groups, w, b, eps, activation == "silu", d_y)
    close(y.detach(), want, x.dtype, units, "y")
    close(grads[0], want_grads[0], x.dtype, units, "dx")
    for name, got, ref, p in zip(("first parameter", "second parameter"), grads[1:], want_grads[1:], leaves[1:]):
        assert got.dtype == p.dtype
        close(got, ref, p.dtype, param_units, name)


MAPS = [  # shape, groups: on the chip in one block, in clusters of 2, 4 and 8, in two passes; odd groups and channels
    ((2, 7, 9, 64), 8), ((1, 1, 1, 32), 4), ((3, 5, 12), 3), ((2, 6), 2), ((1, 40, 41, 24), 24), ((2, 60, 50, 64), 2), ((1, 97, 131, 48), 4),
    ((1, 200, 170, 96), 8), ((1, 181, 203, 40), 5), ((2, 150, 150, 4), 1), ((1, 130, 131, 3), 1), ((2, 14, 14, 1024), 32), ((1, 9, 9, 512), 1),
    ((1, 300, 100, 520), 2),
]


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", MAPS, ids=str)
def test_group_norm(shape, groups, dtype, activation):
    C = shape[-1]
    x = (rand(*shape, scale=1.5) + rand(C, seed=5)).to(dtype)
    check_norm(x, groups, rand(C, seed=1, scale=0.3, shift=1.0), rand(C, seed=2), rand(*shape, dtype=dtype, seed=3), activation)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", [((2, 9, 7, 301), 1), ((1, 5, 1542), 3), ((3, 60, 61, 301), 1), ((1, 1, 2055), 5)], ids=str)
def test_group_norm_of_wide_groups(shape, groups, dtype):
    """More channels a group than a block has threads, and no whole vectors."""
    C = shape[-1]
    x = (rand(*shape, scale=1.5) + rand(C, seed=5)).to(dtype)
    check_norm(x, groups, rand(C, seed=1, scale=0.3, shift=1.0), rand(C, seed=2), rand(*shape, dtype=dtype, seed=3))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_group_norm_parameters(dtype):
    """Of the map's dtype, or one of them, or none."""
    x, d_y = rand(2, 30, 20, 32, dtype=dtype), rand(2, 30, 20, 32, dtype=dtype, seed=3)
    w, b = rand(32, dtype=dtype, seed=1), rand(32, dtype=dtype, seed=2)
    check_norm(x, 4, w, b, d_y)
    check_norm(x, 4, w, None, d_y)
    check_norm(x, 4, None, b, d_y)
    check_norm(x, 4, None, None, d_y, None)


@pytest.mark.parametrize("shape", [(2, 20, 30, 64), (1, 160, 170, 64)], ids=str)
def test_group_norm_far_from_zero(shape):
    """A mean of 300 spreads: variances are taken about means, so the values lose only what they lost as inputs."""
    x = rand(*shape, shift=300.0)
    # x - mean is exact to 2^-24 of 300 spreads, in every element: 1.8e-5, and as much again of the mean
    check_norm(x, 4, None, None, rand(*shape, seed=3), None, units=8)


def test_group_norm_of_one_value():
    x = rand(3, 1, 1, 5, dtype=F32)
    b = rand(5, seed=1)
    y = na.group_norm(x, 5, None, b)
    assert torch.equal(y, b.expand(3, 1, 1, 5))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_views(dtype):
    """An NCHW map permuted to channels last (copied), a slice of the channels, a crop, an odd offset."""
    nchw = rand(2, 32, 11, 13, dtype=dtype).permute(0, 2, 3, 1)
    sliced = rand(2, 11, 13, 96, dtype=dtype)[..., 32:64]
    odd = rand(2, 11, 13, 35, dtype=dtype)[..., 3:]
    crop = rand(2, 15, 16, 32, dtype=dtype)[:, 2:13, 1:14]
    w, b = rand(32, seed=1), rand(32, seed=2)
    for x in (nchw, sliced, odd, crop):
        check_norm(x, 4, w, b, rand(2, 13, 11, 32, dtype=dtype, seed=3).transpose(1, 2))


def test_group_norm_nan_stays_in_its_group():
    x = rand(2, 20, 20, 32, dtype=BF16)
    x[1, 3, 4, 9] = math.nan
    y = na.group_norm(x, 4)
    bad = torch.isnan(y)
    want = torch.zeros_like(bad)
    want[1, :, :, 8:16] = True
    assert torch.equal(bad, want)


def test_group_norm_of_nothing():
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        y = na.group_norm(x, 2, w)
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == gx.shape == x.shape and (gw == 0).all()


def test_group_norm_gradient_against_differences():
    x, w, b, d_y = rand(2, 5, 6, 8), rand(8, seed=1), rand(8, seed=2), rand(2, 5, 6, 8, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(na.group_norm(leaves[0], 2, leaves[1], leaves[2], activation="silu"), leaves, d_y)
    with torch.no_grad():
        for t, g in zip((x, w, b), grads):
            entries = list(range(0, t.numel(), max(1, t.numel() // 12)))
            got = differences(lambda: na.group_norm(x, 2, w, b, activation="silu"), t, d_y, entries, 1e-2)
            assert (got - g.view(-1)[entries].double().cpu()).abs().max() < 5e-3


# ---- rotary positions ---------------------------------------------------------------------------------------------------
def plain_rotary(x, angles, interleaved, inverse=False):
    """x (B, heads, T, C) turned in 64 bits; angles (T, pairs) or (B, 1, T, pairs)."""
    x = x.double()
    half = angles.shape[-1]
    z = torch.polar(torch.ones_like(angles), -angles if inverse else angles)
    low, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        low = torch.view_as_real(torch.complex(low[..., 0::2], low[..., 1::2]) * z).flatten(-2)
    else:
        w = torch.complex(low[..., :half], low[..., half:]) * z
        low = torch.cat((w.real, w.imag), -1)
    return torch.cat((low, rest), -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,N,Nk,T,C,dims", [(1, 1, 1, 1, 8, 8), (2, 4, 2, 37, 64, 64), (1, 3, 3, 100, 128, 64), (2, 5, 1, 11, 48, 12),
                                             (1, 2, 2, 9, 96, 24), (3, 2, 1, 7, 10, 6), (1, 9, 2, 300, 32, 2), (1, 1, 1, 2, 7, 4)])
def test_rotary(B, N, Nk, T, C, dims, dtype, interleaved):
    frequencies = na.rotary_frequencies(dims)
    table = na.rotary_table(torch.arange(T, device=DEV), frequencies)
    angles = torch.arange(T, dtype=torch.float64, device=DEV)[:, None] * frequencies.to(DEV)
    q, k = rand(B, N, T, C, dtype=dtype).requires_grad_(), rand(B, Nk, T, C, dtype=dtype, seed=1).requires_grad_()
    gq, gk = rand(B, N, T, C, dtype=dtype, seed=2), rand(B, Nk, T, C, dtype=dtype, seed=3)
    out = na.rotary(q, k, table, interleaved=interleaved)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for got, x in zip(out, (q, k)):
        close(got.detach(), plain_rotary(x.detach(), angles, interleaved), dtype, 1, "turned")
        assert torch.equal(got.detach()[..., dims:], x.detach()[..., dims:])
    for got, x in zip(grads, (gq, gk)):
        close(got, plain_rotary(x, angles, interleaved, inverse=True), dtype, 1, "gradient")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_rotary_index(kind):
    """A table row for each token; far positions; rows outside the table are NaN, and only their turned channels."""
    rows = 1 << 16
    frequencies = na.rotary_frequencies(32)
    table = na.rotary_table(torch.arange(rows, device=DEV), frequencies)
    q, k = rand(5, 3, 2, 64), rand(5, 1, 2, 64, seed=1)
    index = torch.tensor([[0, rows - 1], [7, 40000], [65535, 1], [-1, 12], [rows, 3]], device=DEV, dtype=kind)
    oq, ok = na.rotary(q, k, table, index)
    angles = index.double()[:, None, :, None] * frequencies.to(DEV)
    outside = (index < 0) | (index >= rows)
    for got, x in ((oq, q), (ok, k)):
        want = plain_rotary(x, angles, False)
        bad = torch.isnan(got)
        assert bad[outside[:, None, :].expand(-1, x.shape[1], -1)][:, :32].all()
        assert not bad[..., 32:].any() and not bad[~outside[:, None, :].expand(-1, x.shape[1], -1)].any()
        keep = ~outside[:, None, :, None].expand_as(x)
        close(got[keep], want[keep], F32, 1, "turned")


def test_rotary_on_grids_and_one_gradient():
    """Axial positions of a grid, views of a packed projection, q alone, a gradient for one of the two only."""
    B, H, W, N, C = 2, 5, 7, 3, 64
    packed = rand(B, H, W, 3, N, C, dtype=BF16)
    q, k, _ = packed.permute(3, 0, 4, 1, 2, 5).unbind(0)
    frequencies = na.rotary_frequencies(32, 100.0)
    table = na.rotary_table(na.rotary_grid(H, W), frequencies)
    rows, cols = torch.meshgrid(torch.arange(H, device=DEV), torch.arange(W, device=DEV), indexing="ij")
    by = frequencies.to(DEV)
    angles = torch.cat((rows.flatten()[:, None] * by, cols.flatten()[:, None] * by), -1)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    oq, ok = na.rotary(q, k, table)
    assert oq.shape == q.shape and ok.shape == k.shape
    close(oq.detach().flatten(2, 3), plain_rotary(q.detach().flatten(2, 3), angles, False), BF16, 1, "q")
    close(ok.detach().flatten(2, 3), plain_rotary(k.detach().flatten(2, 3), angles, False), BF16, 1, "k")
    g = rand(B, N, H, W, C, dtype=BF16, seed=4)
    gq, gk = torch.autograd.grad(ok, (q, k), g, allow_unused=True)
    assert gq is None
    close(gk.flatten(2, 3), plain_rotary(g.flatten(2, 3), angles, False, inverse=True), BF16, 1, "gradient of k")
    alone, none = na.rotary(q, None, table)
    assert none is None and torch.equal(alone, oq)


def test_rotary_table_and_frequencies():
    """Exact angles at far positions, a magnitude, and stretched frequencies against their definition."""
    frequencies = na.rotary_frequencies(64)
    positions = torch.tensor([0, 1, 12345, 1 << 20, (1 << 24) + 1], device=DEV)
    table = na.rotary_table(positions, frequencies, 1.5)
    angles = positions.double()[:, None] * frequencies.to(DEV)
    want = 1.5 * torch.stack((angles.cos(), angles.sin()), -1)
    assert (table.double() - want).abs().max() <= 1.5 * 2.0 ** -24 + 1e-9       # rounded once, of angles up to 2^24 in 64 bits
    assert torch.equal(na.rotary_frequencies(64, stretch=4.0), frequencies / 4)
    scaled = na.rotary_frequencies(64, stretch=8.0, original_length=4096)
    turns = 4096 * frequencies / (2 * math.pi)
    assert torch.equal(scaled[turns >= 32], frequencies[turns >= 32])
    assert torch.allclose(scaled[turns <= 1], frequencies[turns <= 1] / 8, rtol=1e-15)
    assert (scaled <= frequencies).all() and (scaled >= frequencies / 8 * (1 - 1e-15)).all()


# ---- refusals -------------------------------------------------------------------------------------------------------------
def test_refusals():
    q = torch.zeros(2, 4, 8, 32, device=DEV)
    refused = [
        lambda: na.attention(q, q[:, :3], q[:, :3]),                                     # heads that do not divide
        lambda: na.attention(q, q[:1], q[:1]),
        lambda: na.attention(q, q, q[:, :, :4]),
        lambda: na.attention(q, q.half(), q.half()),
        lambda: na.attention(q.double(), q.double(), q.double()),
        lambda: na.attention(q.cpu(), q, q),
        lambda: na.attention(q[0], q[0], q[0]),
        lambda: na.attention(q, q, q, -1.0),
        lambda: na.attention(q, q, q, float("nan")),
        lambda: na.attention(q, q, q, key_lengths=torch.tensor([1, 2])),                 # on the CPU
        lambda: na.attention(q, q, q, key_lengths=torch.tensor([1], device=DEV)),
        lambda: na.attention(q, q, q, key_lengths=torch.tensor([1.0, 2.0], device=DEV)),
        lambda: na.attention_with_lse(q, q, q, path="tensor"),                           # fp32 has no tensor path
        lambda: na.attention(torch.zeros(1, 1, 2, 300, device=DEV), *[torch.zeros(1, 1, 2, 300, device=DEV)] * 2),
        lambda: na.group_norm(q, 5),
        lambda: na.group_norm(q, 0),
        lambda: na.group_norm(q, 4, torch.ones(31, device=DEV)),
        lambda: na.group_norm(q, 4, torch.ones(32, device=DEV, dtype=torch.float64)),
        lambda: na.group_norm(q, 4, torch.ones(32)),
        lambda: na.group_norm(q.half(), 4, torch.ones(32, device=DEV), torch.ones(32, device=DEV).half()),
        lambda: na.group_norm(q, 4, activation="relu"),
        lambda: na.group_norm(q, 4, eps=-1.0),
        lambda: na.group_norm(q.cpu(), 4),
        lambda: na.group_norm(q[0, 0, 0], 4),
        lambda: na.rotary(q, None, torch.zeros(7, 16, 2, device=DEV)),                   # rows for fewer tokens
        lambda: na.rotary(q, None, torch.zeros(8, 17, 2, device=DEV)),                   # more channels than a head has
        lambda: na.rotary(q, None, torch.zeros(8, 16, 2)),
        lambda: na.rotary(q, None, torch.zeros(8, 16, 2, device=DEV).half()),
        lambda: na.rotary(q, q[:, :, :4], torch.zeros(8, 16, 2, device=DEV)),
        lambda: na.rotary(q, None, torch.zeros(8, 16, 2, device=DEV), torch.zeros(2, 7, dtype=torch.int32, device=DEV)),
        lambda: na.rotary(q, None, torch.zeros(8, 16, 2, device=DEV), torch.zeros(2, 8, device=DEV)),
        lambda: na.rotary(q, None, torch.zeros(8, 16, 2, device=DEV, requires_grad=True)),
        lambda: na.rotary_table(torch.arange(4), na.rotary_frequencies(8)),
        lambda: na.rotary_table(torch.zeros(4, 2, device=DEV), torch.zeros(3, 4)),
        lambda: na.rotary_frequencies(7),
        lambda: na.rotary_frequencies(8, stretch=0.0),
    ]
    before = na.launch_count()
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(TypeError):
        na.rotary_table([1, 2], na.rotary_frequencies(8))
    assert na.launch_count() == before


def test_no_second_derivative():
    q = torch.randn(1, 1, 8, 32, device=DEV, requires_grad=True)
    table = na.rotary_table(torch.arange(8, device=DEV), na.rotary_frequencies(32))
    for y in (na.attention(q, q, q), na.group_norm(q, 4), na.rotary(q, None, table)[0]):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(y.sum(), q, create_graph=True)
