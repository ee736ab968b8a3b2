"""The work of the operators that stand around neighborhood attention in a model: group normalisation of
channels-last feature maps, rotary positions on queries and keys, and attention over all keys for the stages
(and the conditioning) where a window is not what is wanted.

A case is one pass through one of them: a training step (forward and backward), an inference forward, or the
single-token form of serving.  Sizes are those of the benchmark and the tests, ragged ones included; ``draw``
spreads further cases over the same ranges.  ``run`` computes the plain form, elementary torch operations in
32 bits, or, where ``own`` is set, calls the package.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# What a drawn case may cost at most: elements of a norm or rotary call, and multiply-adds of one of an
# attention call's products, for 16 bits and for fp32, no more than the largest listed cases; and entries of
# the plain form's score matrix, which it holds a few of.
_MAX_ELEMENTS = 1 << 27
_MAX_MACS = {"fp32": 1 << 32, "bf16": 1 << 38, "fp16": 1 << 38}
_MAX_SCORES = 1 << 31
_MAX_CACHE = 1 << 28


def _norm(op, B, H, W, C, groups, dtype, silu=True):
    return {"op": op, "B": B, "H": H, "W": W, "C": C, "groups": groups, "dtype": dtype, "silu": silu}


def _rotary(op, B, N, Nk, T, C, dims, dtype, interleaved=False, packed=False, table=0):
    """dims: channels that are rotated.  packed: q and k are views of one (B, T, 3, heads, C) projection.
    table: rows of a table that each token picks its own of (0: row t for token t)."""
    return {"op": op, "B": B, "N": N, "Nk": Nk, "T": T, "C": C, "dims": dims, "dtype": dtype,
            "interleaved": interleaved, "packed": packed, "table": table}


def _attention(op, B, N, Nk, Tq, Tk, C, dtype, causal=False, ragged=False, packed=False):
    """Nk: key heads, each shared by N / Nk query heads.  ragged: a number of keys for each batch entry."""
    return {"op": op, "B": B, "N": N, "Nk": Nk, "Tq": Tq, "Tk": Tk, "C": C, "dtype": dtype, "causal": causal,
            "ragged": ragged, "packed": packed}


def listed():
    cases = {
        # smallest: unit-test sized feature map in 32 bits; launches and host time count
        "norm-tiny-fp32-step": _norm("norm_step", 1, 16, 16, 64, 8, "fp32"),
        # deep stage of a vision backbone, training step: a sample fits on the chip
        "norm-stage14-fp16-step": _norm("norm_step", 16, 14, 14, 1024, 32, "fp16"),
        # the benchmark's image-sized grid with its 4 heads of 128 channels, training step
        "norm-side256-bf16-step": _norm("norm_step", 4, 256, 256, 512, 32, "bf16"),
        # inference on an image whose sides fit no tile, no activation
        "norm-ragged-fp16-forward": _norm("norm_forward", 2, 97, 131, 384, 24, "fp16", silu=False),
        # serving: one new token for each of 64 requests, each at its own position, half of a head rotated
        "rotary-token-bf16-forward": _rotary("rotary_forward", 64, 16, 4, 1, 128, 64, "bf16", interleaved=True, table=65536),
        # the benchmark's image-sized grid, q and k sliced out of one projection, training step
        "rotary-side256-bf16-step": _rotary("rotary_step", 4, 4, 4, 65536, 128, 128, "bf16", packed=True),
        # deepest stage: 196 tokens, many heads, q / k / v sliced out of one projection, training step
        "attention-stage14-fp16-step": _attention("attention_step", 16, 16, 16, 196, 196, 64, "fp16", packed=True),
        # the benchmark's small grid with all keys in place of a window, training step
        "attention-side64-bf16-step": _attention("attention_step", 4, 4, 4, 4096, 4096, 128, "bf16"),
        # an image's tokens look at conditioning of different lengths, one of none; shared key heads; training step
        "attention-cross-bf16-step": _attention("attention_step", 8, 16, 4, 3136, 333, 64, "bf16", ragged=True),
        # serving: one new token a request, caches filled to different lengths, shared key heads
        "attention-token-bf16-forward": _attention("attention_forward", 16, 16, 4, 1, 32768, 128, "bf16", causal=True, ragged=True),
        # largest: a long sequence, causal, training step
        "attention-seq16384-bf16-step": _attention("attention_step", 1, 8, 8, 16384, 16384, 128, "bf16", causal=True),
        # the smallest grid of the benchmark in the reference's data type, training step
        "attention-side32-fp32-step": _attention("attention_step", 4, 4, 4, 1024, 1024, 128, "fp32"),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_norm(rng):
    groups = rng.choice([1, 8, 16, 24, 32])
    C = groups * rng.choice([2, 4, 8, 12, 16, 32])
    H = _log_int(rng, 8, 512)
    W = max(8, min(512, round(H * rng.uniform(0.6, 1.7))))
    return _norm(rng.choice(["norm_step", "norm_step", "norm_forward"]), _log_int(rng, 1, 32), H, W, C, groups,
                 rng.choice(list(_DTYPES)), silu=rng.random() < 0.7)


def _draw_rotary(rng):
    Nk = _log_int(rng, 1, 16)
    N = Nk * rng.choice([1, 1, 1, 2, 4])
    C = rng.choice([32, 64, 64, 128, 128, 48, 96])
    dims = rng.choice([C, C, C // 2, C // 4])
    if rng.random() < 0.3:
        return _rotary("rotary_forward", _log_int(rng, 1, 256), N, Nk, 1, C, dims, rng.choice(list(_DTYPES)),
                       interleaved=rng.random() < 0.5, table=_log_int(rng, 1024, 1 << 17))
    return _rotary(rng.choice(["rotary_step", "rotary_step", "rotary_forward"]), _log_int(rng, 1, 32), N, Nk,
                   _log_int(rng, 64, 65536), C, dims, rng.choice(list(_DTYPES)), interleaved=rng.random() < 0.5,
                   packed=N == Nk and rng.random() < 0.5)


def _draw_attention(rng):
    Nk = _log_int(rng, 1, 16)
    N = Nk * rng.choice([1, 1, 1, 2, 4, 8])
    C = rng.choice([32, 64, 64, 64, 128, 128, 128, 48, 96])
    B = _log_int(rng, 1, 32)
    kind = rng.random()
    if kind < 0.25:                                             # serving, a token or a few at a time
        return _attention("attention_forward", B, N, Nk, rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 128, 65536), C,
                          rng.choice(["bf16", "fp16"]), causal=True, ragged=rng.random() < 0.7)
    op = rng.choice(["attention_step", "attention_step", "attention_forward"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "bf16", "fp16"])
    Tq = _log_int(rng, 16, 16384)
    if kind < 0.5:                                              # conditioning of another length than the image
        return _attention(op, B, N, Nk, Tq, _log_int(rng, 7, 2048), C, dtype, ragged=rng.random() < 0.6)
    return _attention(op, B, N, Nk, Tq, Tq, C, dtype, causal=rng.random() < 0.4, packed=N == Nk and rng.random() < 0.4)


def draw(rng):
    while True:
        case = rng.choice([_draw_norm, _draw_rotary, _draw_attention, _draw_attention])(rng)
        kind = case["op"].split("_")[0]
        if kind == "norm":
            fits = 1 << 13 <= case["B"] * case["H"] * case["W"] * case["C"] <= _MAX_ELEMENTS
        elif kind == "rotary":
            fits = 1 << 13 <= case["B"] * case["N"] * case["T"] * case["C"] <= _MAX_ELEMENTS
        else:
            scores = case["B"] * case["N"] * case["Tq"] * case["Tk"]
            fits = (1 << 13 <= scores <= _MAX_SCORES and scores * case["C"] <= _MAX_MACS[case["dtype"]]
                    and case["B"] * case["Nk"] * case["Tk"] * case["C"] <= _MAX_CACHE)
        if fits:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------
def _lengths(case):
    """Keys of each batch entry: from all of them down to none."""
    B, Tk = case["B"], case["Tk"]
    return [Tk - Tk * b // max(B - 1, 1) for b in range(B)] if case["ragged"] else [Tk] * B


def _table(positions, dims):
    """(rows, dims / 2, 2): the cosine and the sine of each position's angle for each pair of channels."""
    frequencies = 10000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    angles = positions.double()[:, None] * frequencies
    return torch.stack((angles.cos(), angles.sin()), -1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, train = case["op"].split("_")[0], case["op"].endswith("step")
    dtype, B, C = _DTYPES[case["dtype"]], case["B"], case["C"]

    def normal(*shape, dtype=dtype, scale=1.0, shift=0.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    state = {"op": case["op"], "train": train}
    if kind == "norm":
        x = normal(B, case["H"], case["W"], C)
        x *= 1.5
        x += normal(C)                                          # channels have means of their own
        state.update(x=x.requires_grad_(train), groups=case["groups"], activation="silu" if case["silu"] else None,
                     weight=normal(C, dtype=torch.float32, scale=0.2, shift=1.0).requires_grad_(train),
                     bias=normal(C, dtype=torch.float32, scale=0.2).requires_grad_(train))
        if train:
            state["d_y"] = normal(B, case["H"], case["W"], C)
        return state

    N, Nk = case["N"], case["Nk"]
    Tq, Tk = (case["T"], case["T"]) if kind == "rotary" else (case["Tq"], case["Tk"])
    if case["packed"]:
        views = normal(B, Tq, 3, N, C).permute(2, 0, 3, 1, 4).unbind(0)     # of one projection
    else:
        views = (normal(B, N, Tq, C), normal(B, Nk, Tk, C), normal(B, Nk, Tk, C))
    state.update(zip("qkv", (t.requires_grad_(train) for t in views)))
    if kind == "rotary":
        state["interleaved"], state["index"] = case["interleaved"], None
        if case["table"]:
            state["index"] = torch.randint(case["table"], (B, Tq), generator=gen, device="cuda", dtype=torch.int32)
        state["table"] = _table(torch.arange(case["table"] or Tq, device="cuda"), case["dims"])
        if train:
            state["d_q"], state["d_k"] = normal(B, N, Tq, C), normal(B, Nk, Tk, C)
        return state
    state.update(scale=C ** -0.5, causal=case["causal"], lengths=None)
    if case["ragged"]:
        state["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    if train:       # the gradient comes back from the output projection, heads last
        state["d_o"] = normal(B, Tq, N, C).permute(0, 2, 1, 3)
    return state


# ---- the package's operators ------------------------------------------------------------------------------------
def _run_own(state):
    import e_natten_b200 as na
    kind = state["op"].split("_")[0]
    if kind == "norm":
        names, leaves, grads = ("y",), (state["x"], state["weight"], state["bias"]), ("d_y",)
        call = lambda: (na.group_norm(state["x"], state["groups"], state["weight"], state["bias"], activation=state["activation"]),)
    elif kind == "rotary":
        names, leaves, grads = ("q", "k"), (state["q"], state["k"]), ("d_q", "d_k")
        call = lambda: na.rotary(state["q"], state["k"], state["table"], state["index"], interleaved=state["interleaved"])
    else:
        names, leaves, grads = ("o",), (state["q"], state["k"], state["v"]), ("d_o",)
        call = lambda: (na.attention(state["q"], state["k"], state["v"], state["scale"], causal=state["causal"],
                                     key_lengths=state["lengths"]),)
    if not state["train"]:
        with torch.no_grad():
            return dict(zip(names, call()))
    outputs = call()
    found = torch.autograd.grad(outputs, leaves, [state[g] for g in grads])
    return {**{n: t.detach() for n, t in zip(names, outputs)}, **{f"grad{i}": g for i, g in enumerate(found)}}


# ---- plain forms ------------------------------------------------------------------------------------------------
def _plain_norm(state):
    x, G = state["x"], state["groups"]
    B, C = x.shape[0], x.shape[-1]
    grouped = lambda t: t.reshape(B, -1, G, C // G)
    whole = lambda t: t.reshape(B, -1, C)
    w, b = state["weight"].reshape(G, C // G), state["bias"].reshape(G, C // G)
    xf = grouped(x.float())
    centred = xf - xf.mean((1, 3), keepdim=True)
    r = (centred.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    xhat = centred * r
    z = xhat * w + b
    s = 1 / (1 + torch.exp(-z)) if state["activation"] else None
    y = z if s is None else z * s
    out = {"y": y.reshape(x.shape).to(x.dtype)}
    if state["train"]:
        dz = grouped(state["d_y"].float())
        if s is not None:
            dz = dz * (s * (1 + z * (1 - s)))
        dxhat = dz * w
        dx = r * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
        out.update(grad0=dx.reshape(x.shape).to(x.dtype), grad1=whole(dz * xhat).sum((0, 1)), grad2=whole(dz).sum((0, 1)))
    return out


def _rotated(x, cos, sin, interleaved):
    """x with its first channels turned by the angles, in the type of x."""
    half = cos.shape[-1]
    xf = x.float()
    turned, rest = xf[..., :2 * half], xf[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _plain_rotary(state):
    table, index = state["table"], state["index"]
    rows = table[:state["q"].shape[2]] if index is None else table[index.long()].unsqueeze(1)
    cos, sin = rows.unbind(-1)
    out = {n: _rotated(state[n], cos, sin, state["interleaved"]) for n in ("q", "k")}
    if state["train"]:      # a gradient turns back
        out.update(grad0=_rotated(state["d_q"], cos, -sin, state["interleaved"]),
                   grad1=_rotated(state["d_k"], cos, -sin, state["interleaved"]))
    return out


def _plain_attention(state):
    q, k, v, scale = state["q"], state["k"], state["v"], state["scale"]
    B, N, Tq, C = q.shape
    Nk, Tk = k.shape[1:3]
    rows = lambda t: t.float().reshape(B * Nk, -1, C)           # of all query heads that share a key head
    back = lambda t, like: t.reshape(like.shape).to(like.dtype)
    lengths = torch.full((B,), Tk, device=q.device) if state["lengths"] is None else state["lengths"].long()
    last = lengths[:, None] + (torch.arange(1 - Tq, 1, device=q.device) if state["causal"] else torch.zeros(Tq, device=q.device))
    hidden = (torch.arange(Tk, device=q.device) >= last[..., None]).repeat_interleave(Nk, 0)[:, None]
    qf, kf, vf = rows(q), rows(k), rows(v)
    s = (qf @ kf.transpose(1, 2)).mul_(scale).view(B * Nk, N // Nk, Tq, Tk).masked_fill_(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0, 1.0)).view(B * Nk, -1, Tk)
    o = p @ vf
    out = {"o": back(o, q)}
    if state["train"]:
        g = rows(state["d_o"])
        dv = p.transpose(1, 2) @ g
        dp = g @ vf.transpose(1, 2)
        ds = dp.sub_((o * g).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out.update(grad0=back(ds @ kf, q), grad1=back(ds.transpose(1, 2) @ qf, k), grad2=back(dv, v))
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}[state["op"].split("_")[0]](state)


# ---- what a pass has to do ----------------------------------------------------------------------------------
def work(case):
    """Each call's inputs read once and its outputs written once (a step is two calls: the forward's inputs
    are read again by the backward); 2 operations per multiply-add over the pairs that the masks leave."""
    kind, train = case["op"].split("_")[0], case["op"].endswith("step")
    esize = 4 if case["dtype"] == "fp32" else 2
    B, C = case["B"], case["C"]
    if kind == "norm":
        t = B * case["H"] * case["W"] * C
        return {"bytes": (5 if train else 2) * t * esize, "flops": (30 if train else 10) * t}
    if kind == "rotary":
        t = B * (case["N"] + case["Nk"]) * case["T"] * C
        rows = B if case["table"] else case["T"]
        calls = 2 if train else 1
        return {"bytes": calls * (2 * t * esize + 4 * rows * case["dims"]), "flops": calls * 3 * t}
    N, Tq = case["N"], case["Tq"]
    lengths = _lengths(case)
    if case["causal"]:                                          # row i of Tq sees length - Tq + 1 + i keys
        pairs = N * sum(sum(range(max(n - Tq + 1, 0), n + 1)) for n in lengths)
    else:
        pairs = N * Tq * sum(lengths)
    t_q, t_k, stat = B * N * Tq * C * esize, case["Nk"] * sum(lengths) * C * esize, 4 * B * N * Tq
    mac = 2.0 * pairs * C
    if not train:
        return {"bytes": 2 * t_q + 2 * t_k, "flops": 2 * mac}
    whole = B * case["Nk"] * case["Tk"] * C * esize             # the gradients of hidden keys are written, too
    return {"bytes": 6 * t_q + 4 * t_k + 2 * whole + 2 * stat, "flops": 7 * mac}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _exact_norm(state):
    x, G = state["x"].detach().double(), state["groups"]
    B, C = x.shape[0], x.shape[-1]
    flat = x.reshape(B, -1, C)
    y, dx = torch.empty_like(flat), torch.empty_like(flat)
    dw, db = x.new_zeros(C), x.new_zeros(C)
    for b in range(B):
        for c in range(0, C, C // G):
            at = slice(c, c + C // G)
            part = flat[b, :, at]
            var, mean = torch.var_mean(part, correction=0)
            root = torch.sqrt(var + 1e-5)
            xhat = (part - mean) / root
            w, bias = state["weight"][at].detach().double(), state["bias"][at].detach().double()
            z = xhat * w + bias
            s = torch.sigmoid(z) if state["activation"] else torch.ones_like(z)
            y[b, :, at] = z * s
            if state["train"]:
                g = state["d_y"].reshape(B, -1, C)[b, :, at].double()
                if state["activation"]:
                    g = g * (s + z * s * (1 - s))
                dw[at] += (g * xhat).sum(0)
                db[at] += g.sum(0)
                g = g * w
                dx[b, :, at] = (g - g.mean() - xhat * (g * xhat).mean()) / root
    out = {"y": y.view_as(x)}
    return {**out, "grad0": dx.view_as(x), "grad1": dw, "grad2": db} if state["train"] else out


def _exact_rotary(state, case):
    half = case["dims"] // 2
    T = state["q"].shape[2]
    frequencies = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    positions = torch.arange(T, device="cuda") if state["index"] is None else state["index"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[..., None] * frequencies)
    turn = turn if state["index"] is None else turn.unsqueeze(1)

    def rotate(x, by):
        x = x.detach().double()
        low, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["interleaved"]:
            low = torch.view_as_real(torch.view_as_complex(low.unflatten(-1, (half, 2)).contiguous()) * by).flatten(-2)
        else:
            z = torch.complex(low[..., :half], low[..., half:]) * by
            low = torch.cat((z.real, z.imag), -1)
        return torch.cat((low, rest), -1)

    out = {n: rotate(state[n], turn) for n in ("q", "k")}
    if state["train"]:
        out.update(grad0=rotate(state["d_q"], turn.conj()), grad1=rotate(state["d_k"], turn.conj()))
    return out


def _exact_attention(state, case):
    """One query head at a time, over the keys that its batch entry has."""
    q, k, v = (state[n].detach() for n in "qkv")
    B, N, Tq, C = q.shape
    shared = N // k.shape[1]
    o, dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, q, k, v))
    for b, length in enumerate(_lengths(case)):
        first = max(Tq - length, 0) if case["causal"] else 0    # rows before it see nothing
        if length == 0 or first == Tq:
            continue
        for n in range(N):
            m = n // shared
            qn, kn, vn = q[b, n, first:].double(), k[b, m, :length].double(), v[b, m, :length].double()
            s = qn @ kn.T * state["scale"]
            if case["causal"]:
                s += torch.full(s.shape, -math.inf, dtype=torch.float64, device="cuda").triu(1 + length - (Tq - first))
            p = torch.softmax(s, -1)
            del s
            o[b, n, first:] = p @ vn
            if state["train"]:
                g = state["d_o"][b, n, first:].double()
                dv[b, m, :length] += p.T @ g
                ds = g @ vn.T
                ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * state["scale"]
                dq[b, n, first:] = ds @ kn
                dk[b, m, :length] += ds.T @ qn
    return {"o": o, "grad0": dq, "grad1": dk, "grad2": dv} if state["train"] else {"o": o}


def exact(case, seed):
    """What ``run`` returns for these inputs, in 64 bits, from the operators' definitions."""
    state = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(state)
    return (_exact_rotary if case["op"].startswith("rotary") else _exact_attention)(state, case)
