"""A small grid transformer that trains on pictures and describes them token by token: windowed attention beside
group normalisation, rotary positions and attention over all keys, as a model would use them.

    PYTHONPATH=. python examples/grid_transformer.py            # trains, then writes out a few tokens

The data are made up: a picture is a wave over a background, and its description counts up from the background's
brightness in steps of the wave's frequency, to a different length for each picture.
"""
from __future__ import annotations

import argparse

import torch
from torch import nn
from torch.nn import functional as F

import e_natten_b200 as na


def heads_of(x, heads):
    """(B, ..., heads C) -> (B, heads, ..., C), a view."""
    x = x.unflatten(-1, (heads, -1))
    return x.movedim(-2, 1)


def tokens_of(x):
    """(B, heads, ..., C) -> (B, ..., heads C)."""
    return x.movedim(1, -2).flatten(-2)


class GroupNorm(nn.Module):
    def __init__(self, channels, groups, activation=None):
        super().__init__()
        self.groups, self.activation = groups, activation
        self.weight, self.bias = nn.Parameter(torch.ones(channels)), nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        return na.group_norm(x, self.groups, self.weight, self.bias, activation=self.activation)


class GridBlock(nn.Module):
    """On a map (B, H, W, channels): a window around each pixel, or all pixels where ``window`` is None."""

    def __init__(self, channels, heads, groups, window):
        super().__init__()
        self.heads, self.window = heads, window
        self.norm, self.qkv, self.out = GroupNorm(channels, groups), nn.Linear(channels, 3 * channels), nn.Linear(channels, channels)
        self.mlp = nn.Sequential(GroupNorm(channels, groups), nn.Linear(channels, 2 * channels), GroupNorm(2 * channels, groups, "silu"),
                                 nn.Linear(2 * channels, channels))

    def forward(self, x, table):
        q, k, v = (heads_of(t, self.heads) for t in self.qkv(self.norm(x)).chunk(3, -1))
        q, k = na.rotary(q, k, table)
        scale = q.shape[-1] ** -0.5
        if self.window is None:
            o = na.attention(q, k, v, scale)
        else:
            o = na.natten2d(q, k, v, self.window, scale=scale)
        x = x + self.out(tokens_of(o))
        return x + self.mlp(x)


class TokenBlock(nn.Module):
    """On tokens (B, T, channels): the tokens before, then the picture.  Key heads are shared by two query heads."""

    def __init__(self, channels, heads):
        super().__init__()
        self.heads, self.key_heads = heads, heads // 2
        half = channels // 2
        self.norms = nn.ModuleList(nn.LayerNorm(channels) for _ in range(3))
        self.qkv, self.out = nn.Linear(channels, channels + 2 * half), nn.Linear(channels, channels)
        self.q_look, self.kv_look, self.out_look = nn.Linear(channels, channels), nn.Linear(channels, 2 * half), nn.Linear(channels, channels)
        self.mlp = nn.Sequential(nn.Linear(channels, 2 * channels), nn.SiLU(), nn.Linear(2 * channels, channels))

    def look(self, picture):
        """Keys and values of the picture's pixels (B, pixels, channels)."""
        return [heads_of(t, self.key_heads) for t in self.kv_look(picture).chunk(2, -1)]

    def forward(self, x, picture, table, lengths=None, cache=None, index=None):
        """``lengths``: tokens of each entry.  Serving: x is one token of each entry, written behind ``cache``, (keys,
        values), at ``index`` (B, 1); lengths then count it."""
        channels = x.shape[-1]
        q, k, v = self.qkv(self.norms[0](x)).split((channels, channels // 2, channels // 2), -1)
        q, k, v = heads_of(q, self.heads), heads_of(k, self.key_heads), heads_of(v, self.key_heads)
        q, k = na.rotary(q, k, table, index)
        scale = q.shape[-1] ** -0.5
        if cache is not None:
            entries = torch.arange(len(x), device=x.device)
            cache[0][entries, :, index[:, 0]] = k[:, :, 0]
            cache[1][entries, :, index[:, 0]] = v[:, :, 0]
            o = na.attention(q, cache[0], cache[1], scale, causal=True, key_lengths=lengths)
        else:                                            # (whole sequences: what lies behind an entry's end sees, and is seen by, nothing else)
            o = na.attention(q, k, v, scale, causal=True)
        x = x + self.out(tokens_of(o))
        q = heads_of(self.q_look(self.norms[1](x)), self.heads)
        x = x + self.out_look(tokens_of(na.attention(q, *picture, scale)))
        return x + self.mlp(self.norms[2](x))


class Describer(nn.Module):
    def __init__(self, side=32, channels=64, heads=4, groups=8, window=7, words=16, most_tokens=12, token_blocks=2):
        super().__init__()
        self.side, self.heads, self.words, self.most_tokens = side, heads, words, most_tokens
        self.embed = nn.Linear(1, channels)
        self.near = GridBlock(channels, heads, groups, window)
        self.merge = nn.Linear(4 * channels, channels)
        self.far = GridBlock(channels, heads, groups, None)
        self.word = nn.Embedding(words + 1, channels)     # the last one begins every description
        self.blocks = nn.ModuleList(TokenBlock(channels, heads) for _ in range(token_blocks))
        self.norm, self.head = nn.LayerNorm(channels), nn.Linear(channels, words)

    def tables(self, device):
        """Rotary tables: both grids', and the tokens'.  (A program keeps them.)"""
        C = self.embed.out_features // self.heads
        axis = na.rotary_frequencies(C // 2, base=100.0)
        return (na.rotary_table(na.rotary_grid(self.side, self.side, device), axis),
                na.rotary_table(na.rotary_grid(self.side // 2, self.side // 2, device), axis),
                na.rotary_table(torch.arange(self.most_tokens, device=device), na.rotary_frequencies(C)))

    def see(self, pictures, tables):
        """Pictures (B, side, side) -> the token blocks' keys and values of the pixels."""
        x = self.near(self.embed(pictures.unsqueeze(-1)), tables[0])
        B, H, W, C = x.shape
        x = self.merge(x.view(B, H // 2, 2, W // 2, 2, C).transpose(2, 3).reshape(B, H // 2, W // 2, 4 * C))
        pixels = self.far(x, tables[1]).flatten(1, 2)
        return [block.look(pixels) for block in self.blocks]

    def forward(self, pictures, words, tables):
        """Logits (B, T, words) of every next word of descriptions (B, T)."""
        seen = self.see(pictures, tables)
        begin = words.new_full((len(words), 1), self.words)
        x = self.word(torch.cat((begin, words[:, :-1]), 1))
        for block, picture in zip(self.blocks, seen):
            x = block(x, picture, tables[2][:x.shape[1]])
        return self.head(self.norm(x))

    @torch.no_grad()
    def describe(self, pictures, tables, lengths, words=None):
        """Logits (B, T, words) and words (B, T), one token at a time, up to each entry's own length; with ``words``
        given, of those."""
        B, T, device = len(pictures), int(lengths.max()), pictures.device
        seen = self.see(pictures, tables)
        caches = [[torch.zeros(B, block.key_heads, T, k.shape[-1], device=device, dtype=k.dtype) for k in picture]
                  for block, picture in zip(self.blocks, seen)]
        last, logits, out = torch.full((B, 1), self.words, device=device), [], []
        for t in range(T):
            index = torch.full((B, 1), t, device=device, dtype=torch.int32)
            have = torch.where(lengths > t, t + 1, 0).int()              # entries that are done look at nothing
            x = self.word(last)
            for block, picture, cache in zip(self.blocks, seen, caches):
                x = block(x, picture, tables[2], have, cache, index)
            logits.append(self.head(self.norm(x)))
            last = logits[-1].argmax(-1) if words is None else words[:, t:t + 1]
            out.append(last)
        return torch.cat(logits, 1), torch.cat(out, 1)


def make_pictures(B, model, generator, device):
    """Pictures, their descriptions, and the descriptions' lengths."""
    T, side = model.most_tokens, model.side
    first = torch.randint(0, model.words, (B, 1), generator=generator)
    step = torch.randint(1, 4, (B, 1), generator=generator)
    lengths = torch.randint(1, T + 1, (B,), generator=generator)
    words = (first + step * torch.arange(T)) % model.words
    at = torch.arange(side) / side * 2 * torch.pi
    pictures = (first / model.words + 0.3 * torch.cos(step * at))[:, :, None].expand(-1, -1, side) + 0.05 * torch.randn(B, side, side, generator=generator)
    return pictures.to(device), words.to(device), lengths.to(device)


def train(model, steps, batch=16, lr=2e-3, dtype=torch.bfloat16, seed=0):
    """Losses of every step."""
    device = next(model.parameters()).device
    generator = torch.Generator().manual_seed(seed)
    tables, losses = model.tables(device), []
    optimizer = torch.optim.AdamW(model.parameters(), lr)
    for _ in range(steps):
        pictures, words, lengths = make_pictures(batch, model, generator, device)
        with torch.autocast("cuda", dtype, enabled=dtype != torch.float32):
            logits = model(pictures, words, tables)
        there = torch.arange(model.most_tokens, device=device) < lengths[:, None]
        loss = F.cross_entropy(logits[there].float(), words[there])
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    options = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    options.add_argument("--steps", type=int, default=200)
    steps = options.parse_args().steps
    torch.manual_seed(0)
    model = Describer().cuda()
    losses = train(model, steps)
    for i in range(0, steps, max(1, steps // 10)):
        print(f"step {i:4d}  loss {losses[i]:.3f}")
    pictures, words, lengths = make_pictures(4, model, torch.Generator().manual_seed(1), "cuda")
    with torch.autocast("cuda", torch.bfloat16):
        _, got = model.describe(pictures, model.tables("cuda"), lengths)
    for b, n in enumerate(lengths.tolist()):
        print("described as", got[b, :n].tolist(), " was", words[b, :n].tolist())


if __name__ == "__main__":
    main()
