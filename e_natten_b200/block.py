"""What stands around neighborhood attention in a model: group normalisation of channels-last feature maps,
rotary positions on queries and keys, and attention over all keys for the stages, and the conditioning, that want
no window.  Differentiable, in float32, bfloat16 and float16, on the caller's stream; like the windowed operators
they run in libna2d.so and have no CPU path.  ``torch.jit.trace`` and dispatch modes record them as operators
of ``torch.ops.e_natten_b200``.

They take the windowed operators' layouts: ``(B, heads, T, C)`` or ``(B, heads, H, W, C)`` queries, keys and
values, strided views of a packed projection among them, and ``(B, ..., C)`` feature maps.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import torch_ext

_ACTIVATIONS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU}
_PATHS = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tensor": _lib.PATH_TENSOR}


# ---- attention over all keys --------------------------------------------------------------------------------
def attention_with_lse(q, k, v, scale=None, causal=False, key_lengths=None, path="auto"):
    """Like :func:`attention` but also returns the (non-differentiable) fp32 row log-sum-exp, ``-inf`` for a row
    that sees no key.  ``path``: "tensor" and "simt" ask for the tensor-core or the CUDA-core kernels."""
    return torch_ext.attention(q, k, v, 1.0 if scale is None else scale, causal, key_lengths, _PATHS[path])


def attention(q, k, v, scale=None, causal=False, key_lengths=None):
    """softmax(scale * q k^T) v over all keys.

    ``q`` is ``(B, heads, T, C)`` or ``(B, heads, H, W, C)``; ``k`` and ``v`` may have another number of tokens,
    and fewer heads: each is then shared by ``heads / key heads`` query heads.  ``scale`` (default: none, as in
    ``natten2d``) multiplies the logits.

    ``key_lengths``, an int32 or int64 tensor of ``(B,)`` on the device, gives each batch entry's number of keys:
    what ``k`` and ``v`` hold beyond is never looked at, and gets gradients of zero.  With ``causal`` the queries
    are the last tokens of the keys' sequence: row ``i`` of ``T`` sees the first ``length - T + 1 + i`` keys, and a
    single query is the newest token of a cache.  A row that sees no key gives zeros.

    A value of ``v`` (``k``, ``q`` or the gradient) that is not finite reaches rows that a causal mask hides it
    from if they lie in the same tile of 128: it meets a weight of zero there.  Rows that see no key, and keys
    beyond a length, get their zeros all the same.

    Scores, weights and sums are float32.  For 16-bit types the weights are rounded to the type for their products
    with ``v`` and with the gradient: ``o`` and the gradient of ``v`` are up to 1.4 times as far off as rounding
    them once puts them.  Head dims go up to 256; ``scale`` is positive.
    """
    return torch_ext.attention(q, k, v, 1.0 if scale is None else scale, causal, key_lengths, _lib.PATH_AUTO)[0]


# ---- group normalisation ----------------------------------------------------------------------------------------
def group_norm(x, num_groups: int, weight=None, bias=None, eps: float = 1e-5, activation: Optional[str] = None):
    """Group normalisation of a channels-last map ``(B, ..., C)``, with ``activation`` (None or "silu") fused in.

    Every batch entry's groups of ``C / num_groups`` consecutive channels are normalised over all their positions.
    ``weight`` and ``bias`` are ``(C,)``, in float32 or the map's dtype.  Statistics are taken in float32.  Maps have
    up to 65535 entries, 16384 channels and 2^29 positions; groups of more than 1024 channels (2048 in 16 bits, 256
    of an odd number of channels) take a block each, however many positions there are.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or 'silu'; got {activation!r}")
    return torch_ext.group_norm(x, num_groups, weight, bias, eps, _ACTIVATIONS[activation])


# ---- rotary positions ---------------------------------------------------------------------------------------------
def rotary_frequencies(dims: int, base: float = 10000.0, *, stretch: float = 1.0, original_length: Optional[int] = None,
                       slow: float = 1.0, fast: float = 32.0) -> torch.Tensor:
    """The ``dims / 2`` angles per position of rotary pairs, float64 on the CPU: ``base ** (-2 i / dims)``.

    ``stretch`` scales them for contexts that many times as long as a model was trained on.  Alone, it divides
    every angle (positions are interpolated).  With ``original_length``, the trained length, it goes by how often a
    pair turns in it: pairs that turn at least ``fast`` times keep their angle, pairs that turn at most ``slow``
    times have it divided, and those between are blended linearly.
    """
    if dims <= 0 or dims % 2:
        raise ValueError(f"dims must be positive and even; got {dims}")
    if not base > 0 or not stretch > 0:
        raise ValueError("base and stretch must be positive")
    frequencies = float(base) ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if original_length is None:
        return frequencies / stretch
    if original_length <= 0 or not fast > slow:
        raise ValueError("original_length must be positive and fast above slow")
    turns = original_length * frequencies / (2 * math.pi)
    kept = ((turns - slow) / (fast - slow)).clamp(0, 1)
    return frequencies * (kept + (1 - kept) / stretch)


def rotary_grid(height: int, width: int, device="cuda") -> torch.Tensor:
    """Positions ``(height * width, 2)`` of a grid's pixels: row and column, for :func:`rotary_table`."""
    rows, cols = torch.meshgrid(torch.arange(height, device=device), torch.arange(width, device=device), indexing="ij")
    return torch.stack((rows.flatten(), cols.flatten()), -1)


def rotary_table(positions: torch.Tensor, frequencies: torch.Tensor, magnitude: float = 1.0) -> torch.Tensor:
    """The table that :func:`rotary` turns by: float32 ``(P, pairs, 2)``, the cosine and the sine of each pair.

    ``positions`` is a CUDA tensor ``(P,)``, or ``(P, axes)`` for positions on several axes; ``frequencies`` is
    ``(pairs,)``, or ``(axes, pairs of an axis)``: pair ``a * n + i`` turns with axis ``a``.  ``(pairs,)`` serves
    every axis of several.  Angles are formed in float64, so that they are exact for long contexts.  ``magnitude``
    multiplies all entries, and with them the turned channels.
    """
    if not isinstance(positions, torch.Tensor) or not isinstance(frequencies, torch.Tensor):
        raise TypeError("positions and frequencies must be tensors")
    if not positions.is_cuda:
        raise ValueError("e_natten_b200 runs on CUDA tensors only (there is no CPU path)")
    if positions.dim() not in (1, 2) or frequencies.dim() not in (1, 2) or frequencies.numel() == 0:
        raise ValueError(f"positions must be (P,) or (P, axes), frequencies (pairs,) or (axes, pairs); "
                         f"got {tuple(positions.shape)} and {tuple(frequencies.shape)}")
    axes = positions.shape[1] if positions.dim() == 2 else 1
    if frequencies.dim() == 1:
        frequencies = frequencies.expand(axes, -1)
    if frequencies.shape[0] != axes:
        raise ValueError(f"frequencies for {frequencies.shape[0]} axes, positions on {axes}")
    at = positions.to(torch.float64).resolve_neg()
    at = at if at.dim() == 2 else at.unsqueeze(-1)
    return torch_ext.rotary_table(at, frequencies.to(positions.device, torch.float64).resolve_neg(), float(magnitude))


def rotary(q, k, table: torch.Tensor, index: Optional[torch.Tensor] = None,
           interleaved: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``q`` and ``k`` (which may be None) with rotary positions, as new dense tensors.

    The first ``2 * pairs`` channels of each head turn by the token's row of ``table`` (see :func:`rotary_table`);
    the others are copied.  Pair ``i`` is channels ``(i, pairs + i)``, or ``(2 i, 2 i + 1)`` where ``interleaved``.
    Token ``t`` has row ``t``, or with ``index``, an int tensor of ``(B, tokens)``, the row that it names: the form
    for serving single tokens.  A row outside the table gives NaN.
    """
    return torch_ext.rotary(q, k, table, index, interleaved)
