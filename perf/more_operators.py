"""The work of the operators for several answers to one prompt: attention over a prefix that answers share and each
answer's own keys, the choice of beam search among beams and words, and the caches that follow their beams.

A case is one pass through one of them: a training step on sampled answers (forward and backward), a step of serving
(one new token an answer, or a few), a choice among all words, a reordering of every layer's caches.  Sizes are
generic, or the example model's; ``draw`` spreads further cases over the same ranges.  ``run`` computes the plain
form, elementary torch operations, or, where ``own`` is set, calls the package.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# What a drawn case may cost at most, no more than the largest listed ones: multiply-adds of one of attention's products
# for 16 bits and for fp32, entries of the plain form's score matrix, values of the caches that attention reads; logits of
# a choice; values of a reordering's caches.
_MAX_MACS = {"fp32": 1 << 31, "bf16": 1 << 36, "fp16": 1 << 36}
_MAX_SCORES = 1 << 29
_MAX_CACHE = 1 << 28
_MAX_LOGITS = 1 << 26
_MAX_MOVED = 1 << 30


def _prefix(op, S, answers, N, Nk, P, Tq, Tk, C, dtype, causal=True, ragged=False, packed=False):
    """S prompts, each with ``answers`` batch entries; P: keys of a prompt; Tk: an answer's own keys (0: none).  ragged: a
    number of prompt keys for each prompt, of own keys for each entry.  packed: q, k, v are views of one projection."""
    return {"op": op, "S": S, "answers": answers, "N": N, "Nk": Nk, "P": P, "Tq": Tq, "Tk": Tk, "C": C, "dtype": dtype,
            "causal": causal, "ragged": ragged, "packed": packed}


def _select(B, K, V, count, dtype, finished=False, masked=False):
    """finished: some beams have ended.  masked: some words are ruled out (logits of minus infinity)."""
    return {"op": "select", "B": B, "K": K, "V": V, "count": count, "dtype": dtype, "finished": finished, "masked": masked}


def _reorder(B, K, alive, layers, heads, T, C, dtype, ragged=False, tokens_first=False):
    """alive: beams of K that others follow.  tokens_first: caches lie as (entries, T, heads, C)."""
    return {"op": "reorder", "B": B, "K": K, "alive": alive, "layers": layers, "heads": heads, "T": T, "C": C, "dtype": dtype,
            "ragged": ragged, "tokens_first": tokens_first}


def listed():
    cases = {
        # the example model's descriptions: two pictures of 256 pixels, two descriptions of each; launches and host time count
        "prefix-tiny-fp32-step": _prefix("prefix_step", 2, 2, 4, 2, 256, 12, 12, 16, "fp32"),
        # training on eight sampled answers to one long prompt
        "prefix-answers-bf16-step": _prefix("prefix_step", 1, 8, 16, 4, 8192, 512, 512, 128, "bf16"),
        # training on four answers to each of four prompts of different lengths, odd sizes, q / k / v of one projection
        "prefix-groups-fp16-step": _prefix("prefix_step", 4, 4, 8, 8, 2048, 333, 333, 64, "fp16", ragged=True, packed=True),
        # serving: 64 requests behind one instruction, one new token each
        "prefix-token-bf16-forward": _prefix("prefix_forward", 1, 64, 32, 8, 16384, 1, 1024, 128, "bf16", ragged=True),
        # beam search: four beams of each of 16 prompts, one new token each
        "prefix-beams-bf16-forward": _prefix("prefix_forward", 16, 4, 16, 4, 8192, 1, 256, 128, "bf16", ragged=True),
        # a few drafted tokens of each of 24 requests
        "prefix-drafts-fp16-forward": _prefix("prefix_forward", 1, 24, 16, 4, 30011, 5, 700, 64, "fp16", ragged=True),
        # the example model's words
        "select-tiny-fp32": _select(4, 4, 16, 4, "fp32"),
        # ordinary vocabulary, twice as many candidates as beams, so that ended ones can be set aside
        "select-ordinary-bf16": _select(16, 4, 32768, 8, "bf16"),
        # odd sizes, beams that have ended, words that are ruled out
        "select-odd-fp16": _select(7, 5, 100003, 10, "fp16", finished=True, masked=True),
        # largest: many requests, large vocabulary
        "select-large-fp32": _select(64, 8, 131072, 8, "fp32"),
        # the example model's caches
        "reorder-tiny-fp32": _reorder(4, 4, 2, 2, 2, 12, 16, "fp32"),
        # largest: every layer's keys and values of 32 beams at different lengths
        "reorder-large-bf16": _reorder(8, 4, 2, 8, 8, 2048, 128, "bf16", ragged=True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_prefix(rng):
    S = rng.choice([1, 1, 1, 2, 4, _log_int(rng, 1, 32)])
    answers = _log_int(rng, 1, 64)
    Nk = _log_int(rng, 1, 16)
    N = Nk * rng.choice([1, 1, 2, 4, 4, 8])
    C = rng.choice([32, 64, 64, 128, 128, 128, 48, 96])
    P = _log_int(rng, 64, 32768)
    ragged = rng.random() < 0.6
    if rng.random() < 0.55:                                     # serving, a token or a few at a time; sometimes the prompt alone
        Tq = rng.choice([1, 1, 1, 2, 5])
        Tk = 0 if rng.random() < 0.15 else _log_int(rng, 8, 4096)
        return _prefix("prefix_forward", S, answers, N, Nk, P, Tq, Tk, C, rng.choice(["bf16", "fp16"]), ragged=ragged)
    T = _log_int(rng, 12, 2048)
    return _prefix(rng.choice(["prefix_step", "prefix_step", "prefix_forward"]), S, answers, N, Nk, P, T, T, C,
                   rng.choice(["fp32", "bf16", "bf16", "bf16", "fp16"]), causal=rng.random() < 0.85, ragged=ragged,
                   packed=N == Nk and rng.random() < 0.5)


def _draw_select(rng):
    K = _log_int(rng, 1, 16)
    V = _log_int(rng, 16, 200000)
    count = min(K * V, rng.choice([K, K, 2 * K]))
    return _select(_log_int(rng, 1, 256), K, V, count, rng.choice(list(_DTYPES)), finished=rng.random() < 0.4,
                   masked=rng.random() < 0.3)


def _draw_reorder(rng):
    K = _log_int(rng, 2, 16)
    return _reorder(_log_int(rng, 1, 32), K, rng.randint(1, K), _log_int(rng, 1, 16), _log_int(rng, 1, 16), _log_int(rng, 12, 8192),
                    rng.choice([16, 32, 48, 64, 96, 128, 128]), rng.choice(list(_DTYPES)), ragged=rng.random() < 0.6,
                    tokens_first=rng.random() < 0.3)


def draw(rng):
    while True:
        case = rng.choice([_draw_prefix, _draw_prefix, _draw_select, _draw_reorder])(rng)
        if case["op"] == "select":
            fits = case["B"] * case["K"] * case["V"] <= _MAX_LOGITS
        elif case["op"] == "reorder":
            values = 2 * case["layers"] * case["B"] * case["K"] * case["heads"] * case["T"] * case["C"]
            fits = 1 << 12 <= values <= (_MAX_MOVED >> (case["dtype"] == "fp32"))
        else:
            B = case["S"] * case["answers"]
            scores = B * case["N"] * case["Tq"] * (case["P"] + case["Tk"])
            values = case["Nk"] * (case["S"] * case["P"] + B * case["Tk"]) * case["C"]
            fits = scores <= _MAX_SCORES and scores * case["C"] <= _MAX_MACS[case["dtype"]] and values <= _MAX_CACHE
        if fits:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------
def _spread(most, least, n):
    """n lengths from ``most`` down to ``least``."""
    return [most - (most - least) * i // max(n - 1, 1) for i in range(n)]


def _prompt_lengths(case):
    return _spread(case["P"], case["P"] // 3, case["S"]) if case["ragged"] else [case["P"]] * case["S"]


def _own_lengths(case):
    """Own keys of each entry: a training step's answers have at least a token, a cache at least the new ones."""
    B = case["S"] * case["answers"]
    if not case["ragged"]:
        return [case["Tk"]] * B
    least = min(case["Tk"], case["Tq"]) if case["Tq"] < case["Tk"] else min(case["Tk"], 1)
    return _spread(case["Tk"], least, B)


def _cache_lengths(case):
    """Tokens of each entry, a group of beams at a time."""
    groups = _spread(case["T"], max(1, case["T"] // 4), case["B"]) if case["ragged"] else [case["T"]] * case["B"]
    return [n for n in groups for _ in range(case["K"])]


def _parents(case, gen):
    """(B, K): each entry follows one of ``alive`` beams, all of which are followed, none of them (where there are two) itself."""
    K, alive, rows = case["K"], case["alive"], []
    for _ in range(case["B"]):
        while True:
            chosen = torch.randperm(K, generator=gen)[:alive]
            row = chosen[torch.arange(K) % alive][torch.randperm(K, generator=gen)]
            if alive == 1 or not (row == torch.arange(K)).any():
                break
        rows.append(row)
    return torch.stack(rows)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    state = {"op": case["op"].split("_")[0], "train": case["op"].endswith("step")}
    if state["op"] == "select":
        B, K, V = case["B"], case["K"], case["V"]
        logits = normal(B, K, V, scale=3.0)
        state["finished"] = None
        if case["masked"]:
            logits[..., torch.randint(V, (max(1, V // 16),), generator=gen, device="cuda")] = -math.inf
        if case["finished"]:
            state["finished"] = torch.rand((B, K), generator=gen, device="cuda") < 0.3
        state.update(logits=logits, scores=normal(B, K, dtype=torch.float32, scale=2.0) - 12.0, count=case["count"], end=V - 1)
        return state
    if state["op"] == "reorder":
        entries, heads, T, C = case["B"] * case["K"], case["heads"], case["T"], case["C"]
        shape = (entries, T, heads, C) if case["tokens_first"] else (entries, heads, T, C)
        caches = [normal(*shape) for _ in range(2 * case["layers"])]
        state["caches"] = [c.transpose(1, 2) for c in caches] if case["tokens_first"] else caches
        state["parents"] = _parents(case, torch.Generator().manual_seed(seed)).to("cuda")
        state["lengths"] = torch.tensor(_cache_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
        return state
    S, N, Nk, P, Tq, Tk, C, train = *(case[n] for n in ("S", "N", "Nk", "P", "Tq", "Tk", "C")), state["train"]
    B = S * case["answers"]
    if case["packed"]:
        views = normal(B, Tq, 3, N, C).permute(2, 0, 3, 1, 4).unbind(0)
    else:
        views = (normal(B, N, Tq, C), *((normal(B, Nk, Tk, C), normal(B, Nk, Tk, C)) if Tk else (None, None)))
    state.update(zip(("q", "k", "v"), views))
    state.update(pk=normal(S, Nk, P, C), pv=normal(S, Nk, P, C), scale=C ** -0.5, causal=case["causal"], lengths=None, prompt_lengths=None)
    if train:
        for n in ("q", "k", "v", "pk", "pv"):
            state[n] = state[n].detach().requires_grad_()
        state["d_o"] = normal(B, Tq, N, C).permute(0, 2, 1, 3)      # comes back from the output projection, heads last
    if case["ragged"]:
        state["prompt_lengths"] = torch.tensor(_prompt_lengths(case), device="cuda", dtype=torch.int32)
        if Tk:
            state["lengths"] = torch.tensor(_own_lengths(case), device="cuda", dtype=torch.int32)
    return state


# ---- the package's operators ------------------------------------------------------------------------------------
def _run_own(state):
    import e_natten_b200 as na
    if state["op"] == "select":
        scores, parents, words = na.beam_select(state["logits"], state["scores"], state["count"], finished=state["finished"], end=state["end"])
        return {"scores": scores, "parents": parents, "words": words}
    if state["op"] == "reorder":
        na.beam_reorder(state["caches"], state["parents"], state["lengths"])
        return state["caches"]
    call = lambda: na.prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["scale"], causal=state["causal"],
                                       key_lengths=state["lengths"], prefix_lengths=state["prompt_lengths"])
    if not state["train"]:
        with torch.no_grad():
            return {"o": call()}
    o = call()
    found = torch.autograd.grad(o, [state[n] for n in ("q", "pk", "pv", "k", "v")], state["d_o"])
    return {"o": o.detach(), **{n: g for n, g in zip(("dq", "dpk", "dpv", "dk", "dv"), found)}}


# ---- plain forms ------------------------------------------------------------------------------------------------
def _plain_prefix(state):
    """Scores against the prompt for all answers at once, and against each answer's own keys, under one softmax."""
    q, pk, pv, k, v, scale = (state[n] for n in ("q", "pk", "pv", "k", "v", "scale"))
    B, N, Tq, C = q.shape
    S, Nk, P = pk.shape[:3]
    A, G = B // S, N // Nk
    # rows of all answers that share a key head of the prompt, (S, Nk, A G Tq, C), and of one answer's, (B, Nk, G Tq, C)
    joint = lambda t: t.float().reshape(S, A, Nk, G * Tq, -1).transpose(1, 2).reshape(S, Nk, A * G * Tq, -1)
    apart = lambda t: t.reshape(S, Nk, A, G * Tq, -1).transpose(1, 2).reshape(B, Nk, G * Tq, -1)
    dev = q.device
    qf, pkf, pvf = joint(q), pk.float(), pv.float()
    s0 = (qf @ pkf.transpose(2, 3)).mul_(scale)
    if state["prompt_lengths"] is not None:
        s0.masked_fill_((torch.arange(P, device=dev) >= state["prompt_lengths"][:, None].long())[:, None, None], -math.inf)
    top = s0.amax(-1, keepdim=True)
    if k is not None:
        Tk = k.shape[2]
        kf, vf = k.float(), v.float()
        s1 = (apart(qf) @ kf.transpose(2, 3)).mul_(scale)
        lengths = torch.full((B,), Tk, device=dev) if state["lengths"] is None else state["lengths"].long()
        seen = lengths[:, None] + (torch.arange(1 - Tq, 1, device=dev) if state["causal"] else torch.zeros(Tq, dtype=torch.long, device=dev))
        hidden = (torch.arange(Tk, device=dev) >= seen[..., None]).repeat(1, G, 1)[:, None]
        s1 = s1.masked_fill_(hidden, -math.inf)
        top = torch.maximum(top, joint(s1.amax(-1, keepdim=True)))
    top = top.masked_fill(top == -math.inf, 0.0)
    p0 = s0.sub_(top).exp_()
    total = p0.sum(-1, keepdim=True)
    if k is not None:
        p1 = s1.sub_(apart(top)).exp_()
        total = total + joint(p1.sum(-1, keepdim=True))
    total = total.masked_fill(total == 0, 1.0)
    p0 = p0.div_(total)
    o = p0 @ pvf
    if k is not None:
        p1 = p1.div_(apart(total))
        o = o + joint(p1 @ vf)
    back = lambda t: apart(t).reshape(q.shape).to(q.dtype)
    out = {"o": back(o)}
    if state["train"]:
        g = joint(state["d_o"])
        delta = (o * g).sum(-1, keepdim=True)
        ds0 = (g @ pvf.transpose(2, 3)).sub_(delta).mul_(p0).mul_(scale)
        ds1 = (apart(g) @ vf.transpose(2, 3)).sub_(apart(delta)).mul_(p1).mul_(scale)
        dq = ds0 @ pkf + joint(ds1 @ kf)
        out.update(dq=back(dq), dpk=(ds0.transpose(2, 3) @ qf).to(pk.dtype), dpv=(p0.transpose(2, 3) @ g).to(pv.dtype),
                   dk=(ds1.transpose(2, 3) @ apart(qf)).to(k.dtype), dv=(p1.transpose(2, 3) @ apart(g)).to(v.dtype))
    return out


def _plain_select(state):
    """Each beam's best words by (logit, lowest word), as whole numbers that order so; then the beams' together.  Sums of
    the exponentials, and the scores that candidates of different beams are ordered by, are in 64 bits."""
    logits, count = state["logits"], state["count"]
    B, K, V = logits.shape
    x = logits.float()
    bits = x.view(torch.int32).long()
    keys = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)).bitwise_left_shift_(32).sub_(torch.arange(V, device=x.device))
    most = min(count, V)
    words = (-torch.topk(keys, most, dim=-1).values).bitwise_and_(0xffffffff)
    del keys
    top = x.amax(-1, keepdim=True)
    total = (x - top).double().exp_().sum(-1, keepdim=True)
    scores = state["scores"].double()[..., None] + (x.gather(-1, words).double() - (top.double() + total.log()))
    if state["finished"] is not None:
        ended = state["finished"][..., None]
        first = torch.arange(most, device=x.device) == 0
        scores = torch.where(ended, torch.where(first, state["scores"].double()[..., None], -math.inf), scores)
        words = torch.where(ended & first, state["end"], words)
        scores = torch.where(ended & ~first, -math.inf, scores)
    order = (torch.arange(K, device=x.device)[:, None] * V + words).flatten(1)
    by_index = order.argsort(-1)
    flat = scores.flatten(1).gather(-1, by_index)
    best = flat.argsort(stable=True, dim=-1, descending=True)[:, :count]
    found = flat.gather(-1, best)
    order = order.gather(-1, by_index.gather(-1, best)).masked_fill(found == -math.inf, 0)
    return {"scores": found.float(), "parents": order // V, "words": order % V}


def _plain_reorder(state):
    caches, parents, lengths = state["caches"], state["parents"], state["lengths"]
    B, K = parents.shape
    source = (parents + K * torch.arange(B, device=parents.device)[:, None]).flatten()
    for cache in caches:
        moved = cache[source]
        if lengths is not None:
            there = torch.arange(cache.shape[2], device=cache.device) < lengths[source][:, None]
            moved = torch.where(there[:, None, :, None], moved, cache)
        cache.copy_(moved)
    return caches


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"prefix": _plain_prefix, "select": _plain_select, "reorder": _plain_reorder}[state["op"]](state)


# ---- what a pass has to do ----------------------------------------------------------------------------------
def work(case):
    """Each call's inputs read once and its outputs written once (a step is two calls); 2 operations a multiply-add over
    the pairs that the masks leave.  A reordering reads each beam that others follow, and writes each entry that follows another."""
    esize = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "select":
        B, K = case["B"], case["K"]
        return {"bytes": B * K * (case["V"] * esize + 4) + 20 * B * case["count"], "flops": 4.0 * B * K * case["V"]}
    if case["op"] == "reorder":
        K, alive = case["K"], case["alive"]
        entry = 2 * case["layers"] * case["heads"] * case["C"] * esize * sum(_cache_lengths(case)[::K])      # of one beam a group
        return {"bytes": entry * (alive + (K - 1 if alive == 1 else K)), "flops": 0}
    N, Nk, Tq, C, S, A = (case[n] for n in ("N", "Nk", "Tq", "C", "S", "answers"))
    B, prompts, lengths = S * A, _prompt_lengths(case), _own_lengths(case)
    pairs = N * Tq * A * sum(prompts)
    if case["causal"]:                                          # row i of Tq sees the first length - Tq + 1 + i own keys
        pairs += N * sum(sum(range(max(n - Tq + 1, 0), n + 1)) for n in lengths)
    else:
        pairs += N * Tq * sum(lengths)
    t_q, t_k, stat = B * N * Tq * C * esize, Nk * (sum(prompts) + sum(lengths)) * C * esize, 4 * B * N * Tq
    mac = 2.0 * pairs * C
    if case["op"] == "prefix_forward":
        return {"bytes": 2 * t_q + 2 * t_k, "flops": 2 * mac}
    whole = Nk * (S * case["P"] + B * case["Tk"]) * C * esize
    return {"bytes": 6 * t_q + 4 * t_k + 2 * whole + 2 * stat, "flops": 7 * mac}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _exact_prefix(state, case):
    """Entry by entry and key head by key head, over the keys that the entry sees, one behind the other."""
    q, pk, pv, k, v = (state[n].detach() if state[n] is not None else None for n in ("q", "pk", "pv", "k", "v"))
    B, N, Tq, C = q.shape
    shared, A = N // pk.shape[1], case["answers"]
    prompts, lengths = _prompt_lengths(case), _own_lengths(case)
    new = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    o = new(q)
    if state["train"]:
        dq, dpk, dpv, dk, dv = (new(t) for t in (q, pk, pv, k, v))
    for b in range(B):
        s, length, prompt = b // A, lengths[b], prompts[b // A]
        if length + prompt == 0:
            continue
        bias = torch.zeros(Tq, prompt + length, dtype=torch.float64, device="cuda")
        if case["causal"] and length:
            last = length - Tq + torch.arange(Tq, device="cuda")
            bias[:, prompt:] = torch.where(torch.arange(length, device="cuda") <= last[:, None], 0.0, -math.inf)
        for m in range(pk.shape[1]):
            keys, values = pk[s, m, :prompt].double(), pv[s, m, :prompt].double()
            if length:
                keys, values = torch.cat((keys, k[b, m, :length].double())), torch.cat((values, v[b, m, :length].double()))
            heads = slice(m * shared, (m + 1) * shared)
            logits = q[b, heads].double() @ keys.T * state["scale"] + bias
            p = torch.softmax(logits, -1)
            if prompt == 0:
                p = torch.nan_to_num(p)
            o[b, heads] = p @ values
            if not state["train"]:
                continue
            g = state["d_o"][b, heads].double()
            w = g @ values.T
            ds = p * (w - (p * w).sum(-1, keepdim=True)) * state["scale"]
            dq[b, heads] = ds @ keys
            by_key, by_value = (ds.transpose(1, 2) @ q[b, heads].double()).sum(0), (p.transpose(1, 2) @ g).sum(0)
            dpk[s, m, :prompt] += by_key[:prompt]
            dpv[s, m, :prompt] += by_value[:prompt]
            dk[b, m, :length] += by_key[prompt:]
            dv[b, m, :length] += by_value[prompt:]
    return {"o": o, "dq": dq, "dpk": dpk, "dpv": dpv, "dk": dk, "dv": dv} if state["train"] else {"o": o}


def _exact_select(state):
    """All beams' words in one line, sorted."""
    logits, count = state["logits"], state["count"]
    B, K, V = logits.shape
    scores, parents, words = [], [], []
    for b in range(B):
        line = torch.log_softmax(logits[b].double(), -1) + state["scores"][b, :, None].double()
        if state["finished"] is not None:
            for i in range(K):
                if state["finished"][b, i]:
                    line[i] = -math.inf
                    line[i, state["end"]] = state["scores"][b, i].double()
        found, at = torch.sort(line.flatten(), descending=True, stable=True)
        found, at = found[:count], torch.where(found[:count] > -math.inf, at[:count], 0)     # (no candidate: beam 0, word 0)
        scores.append(found)
        parents.append(torch.div(at, V, rounding_mode="floor"))
        words.append(at % V)
    return {"scores": torch.stack(scores), "parents": torch.stack(parents), "words": torch.stack(words)}


def _exact_reorder(state, case):
    K = case["K"]
    out = [c.double() for c in state["caches"]]
    lengths = _cache_lengths(case)
    for e, parent in enumerate(state["parents"].flatten().tolist()):
        source = e // K * K + parent
        for cache, was in zip(out, state["caches"]):
            cache[e, :, :lengths[source]] = was[source, :, :lengths[source]].double()
    return out


def exact(case, seed):
    """What ``run`` returns for these inputs, in 64 bits, from the operators' definitions."""
    state = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(state)
    return _exact_reorder(state, case) if case["op"] == "reorder" else _exact_prefix(state, case)
