"""Several answers to one prompt: attention over a prefix that answers share and each answer's own keys, the choice of
beam search among beams and words, and caches that follow their beams.

They stand beside :func:`~e_natten_b200.attention`, in its layouts, types and manners: ``(B, heads, T, C)`` or
``(B, heads, H, W, C)`` queries, keys and values, on the caller's stream, in libna2d.so, with no CPU path.  The answers
to a prompt lie next to one another in the batch: entry ``g * K + i`` is answer ``i`` of prompt ``g``.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import torch_ext
from .block import _PATHS


# ---- attention over a prefix ------------------------------------------------------------------------------------
def prefix_attention_with_lse(q, prefix_k, prefix_v, k=None, v=None, scale=None, causal=False, key_lengths=None, prefix_lengths=None, path="auto"):
    """Like :func:`prefix_attention` but also returns the (non-differentiable) fp32 row log-sum-exp over the prefix's and the
    own keys, ``-inf`` for a row that sees no key.  ``path``: "tensor" and "simt" ask for the tensor-core or the CUDA-core
    kernels."""
    return torch_ext.prefix_attention(q, prefix_k, prefix_v, k, v, 1.0 if scale is None else scale, causal, key_lengths, prefix_lengths, _PATHS[path])


def prefix_attention(q, prefix_k, prefix_v, k=None, v=None, scale=None, causal=False, key_lengths=None, prefix_lengths=None):
    """softmax(scale * q [prefix_k; k]^T) [prefix_v; v]: attention over keys that entries share and their own.

    ``q`` is ``(B, heads, T, C)`` or ``(B, heads, H, W, C)``.  ``prefix_k`` and ``prefix_v`` are ``(S, key heads, P, C)``: S
    prefixes, each shared by the ``B / S`` entries that follow one another and read once for all of them.  ``k`` and ``v``,
    ``(B, key heads, Tk, C)``, are the entries' own keys; without them there is the prefix alone.  ``key heads`` divides
    ``heads``, as in :func:`attention`.

    ``prefix_lengths``, of ``(S,)``, and ``key_lengths``, of ``(B,)``, int32 or int64 on the device, give the numbers of keys that are
    there; what is stored beyond is never looked at, and gets gradients of zero.  Every row sees all of its prefix.  With
    ``causal`` the queries are the last tokens of the own keys' sequence: row ``i`` of ``T`` sees the first
    ``length - T + 1 + i`` own keys.  A row that sees no key gives zeros.

    Gradients of the prefix are sums over its entries, those of q sums over both kinds of keys, formed in float32; the same
    call gives the same bits.  Values that are not finite, roundings, head dims and ``scale`` are as in :func:`attention`.
    """
    return torch_ext.prefix_attention(q, prefix_k, prefix_v, k, v, 1.0 if scale is None else scale, causal, key_lengths, prefix_lengths,
                                      _lib.PATH_AUTO)[0]


# ---- beam search --------------------------------------------------------------------------------------------------
def beam_select(logits, scores, count: Optional[int] = None, finished=None, end: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``count`` best continuations of each entry's beams: ``(scores, parents, words)``, each ``(B, count)``.

    ``logits`` is ``(B, beams, words)`` in float32, bfloat16 or float16, ``scores`` the float32 ``(B, beams)`` worths so far.  Beam ``i``
    followed by word ``w`` is worth ``scores[i] + log_softmax(logits[i])[w]``; the best come first, of equal ones the lowest
    beam, then the lowest word.  ``count`` defaults to the number of beams.  Returned scores are float32, parents (beams) and
    words int64.

    ``finished``, a bool tensor of ``(B, beams)``, marks beams that have ended: such a beam has one candidate, itself, with word
    ``end`` at its score, and its logits are not looked at.  A word whose logit is ``-inf`` is no candidate.  A beam whose score
    is not finite has none (scores of ``-inf`` for all beams but one start a search from one prompt), nor has a beam with a
    logit of NaN or ``+inf``.  Places that are left over have score ``-inf``, parent 0 and word 0.

    Exponentials are float32: a worth is off by less than ``2 ** -16`` (by up to ``2 ** -20`` in rows that were made to be hard), so
    that those of different beams that are nearer to one another than ``2 ** -15`` may come in either order; equal rows of logits have
    equal worths.

    Up to 32 beams, 64 candidates and 2^24 words.  Not differentiable: what has a tangent is refused.
    """
    return torch_ext.beam_select(logits, scores, scores.shape[-1] if count is None else count, finished, end)


def beam_reorder(caches: Union[torch.Tensor, Sequence[torch.Tensor]], parents: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> None:
    """Caches follow their beams, in place: entry ``g * K + i`` becomes what entry ``g * K + parents[g, i]`` was.

    ``parents`` is an int32 or int64 tensor of ``(B, K)``, as :func:`beam_select` returns it.  ``caches`` is a tensor or a sequence of
    them, of any types and sizes, with ``B * K`` entries each: ``(entries, heads, tokens, C)`` with any strides that give each
    element its own place (channels contiguous), or contiguous of any shape.  All entries move at once, whichever follow which, and
    without a second copy of the cache; an entry that is its own parent costs nothing.  A parent outside ``[0, K)`` leaves its
    entry as it is.

    ``lengths``, an int32 or int64 tensor with a number for each entry, says how many tokens each holds: an entry gets its
    parent's, and what is stored behind those stays as it was.  (Lengths themselves do not move: ``lengths.view(B, K).gather(1,
    parents)`` are the new ones.)

    Several caches move one after the other in effect: one that is given twice moves twice.  All are checked
    before one moves; parents and lengths that are among them are taken as they were.  Up to 32 beams.  Not differentiable: what has a tangent is refused.
    """
    torch_ext.beam_reorder([caches] if isinstance(caches, torch.Tensor) else list(caches), parents, lengths)
