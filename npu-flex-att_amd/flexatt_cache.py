"""Serving over a K/V cache on gfx950: new tokens into the cache, attention of a
tree of drafted tokens over it, the attention weight its keys have received, and
eviction by that weight.  No counterpart in the reference, which keeps no cache.

A cache is a pair of [B, Hkv, C, D] tensors (any strides a kernel can read in
place: innermost stride 1, rows on 16-byte boundaries) with ``lengths``, int32 [B]
on the device: the rows of each sequence that are in use.  ``lengths`` stays on the
device, so every call can be captured into a graph and replayed as the cache grows.
A cache of other strides is refused where it is written; where it is only read, the
call copies it whole, every time (tree_attention also one with rows 64 MB or more
apart).

  rotary_append(...)          query' and the cache rows of new tokens, in one kernel
  tree_attention(...)         drafted tokens (or one new token) over cache and tree
  attention_weight_sums(...)  sum over the query rows of the softmax weights, per key
  evict_cache(...)            the rows worth keeping, copied to a smaller cache

None of them is differentiable: a tensor that carries a tangent, or with gradients
on one that requires them, is refused.  Nor can they be traced (``make_fx``, export,
fake tensors); ``torch.compile`` breaks its graph at them.
"""
from __future__ import annotations

import flexatt_lib as _lib

__all__ = ["rotary_append", "tree_attention", "attention_weight_sums", "evict_cache"]


def rotary_append(query, key, value, key_cache, value_cache, lengths, inv_freq, positions=None, interleaved=False,
                  magnitude=1.0):
    """Put new tokens into the cache; returns ``query'``.

    ``query`` [B, Hq, S, D], ``key`` / ``value`` [B, Hkv, S, D]: the tokens behind the
    cached ones.  Rows ``lengths[b] + s`` of ``key_cache`` / ``value_cache`` receive the
    rotated key and the value of token ``s``, and ``query'`` is the rotated query, as
    :func:`flexatt_rotary.rotary_embedding` gives them; ``positions`` (int32 or int64
    [S] or [B, S]) defaults to the rows' numbers.  ``inv_freq=None`` rotates nothing
    and returns a copy of the query.  A row outside the cache is not written.  A query
    without heads puts keys and values into the cache alone.  The new tokens, the key
    cache and the value cache share no memory.
    ``lengths`` is read, not changed.
    """
    return _lib.native().rotary_append(query, key, value, key_cache, value_cache, lengths, inv_freq, positions,
                                       interleaved, magnitude)


def tree_attention(query, key_cache, value_cache, lengths, tree_mask=None, sliding_window=0, depths=None, scale=None,
                   soft_cap=0.0, return_lse=False):
    """Attention of ``T`` drafted tokens per sequence over its cache and over each
    other; returns ``O`` or ``(O, LSE)``.

    ``query`` [B, Hq, T, D].  The cache holds ``lengths[b]`` cached tokens, which each
    drafted token sees, and behind them the drafted tokens' own keys and values (rows
    ``lengths[b] .. lengths[b] + T - 1``, as :func:`rotary_append` writes them), of
    which token ``t`` sees those with ``tree_mask[t][u]`` set: a bool or integer [T, T]
    or [B, T, T], itself and its ancestors for a tree; None is a chain (``u <= t``).
    One token per sequence with no mask is ordinary decoding.  Rows behind those are
    not read; values of rows a token does not see are multiplied by 0, so they must be
    finite.

    ``sliding_window`` W keeps cached token ``j`` for drafted token ``t`` where
    ``lengths[b] + depths[b][t] - j <= W``; ``depths`` (int32 [T] or [B, T], 0 for a
    token directly behind the cached ones) defaults to ``t`` for a chain and must be
    given with a mask.  Within the tree the mask alone decides.  ``scale`` and
    ``soft_cap`` as in ``npu_flash_attention_forward``, and so are ``O`` (in
    ``query``'s dtype and layout), ``LSE`` (fp32 [B, Hq, T], natural log) and a token
    without keys (0 and -inf).  A sequence whose ``lengths[b] + T`` rows do not fit the
    cache, which only the device knows, gets NaN.
    """
    return _lib.native().tree_attention(query, key_cache, value_cache, lengths, tree_mask, sliding_window, depths, scale,
                                        soft_cap, return_lse)


def attention_weight_sums(query, key, lse, causal=False, query_start=0, lengths=None, sliding_window=0, scale=None,
                          soft_cap=0.0, into=None):
    """The attention weight each key has received from the query rows: fp32
    [B, Hkv, Skv], summed over the query heads that share a KV head.

    ``query`` [B, Hq, Sq, D], ``key`` [B, Hkv, Skv, D] (a cache, or the keys of the
    call) and the ``lse`` fp32 [B, Hq, Sq] of the attention they took part in
    (``npu_flash_attention_forward``, ``tree_attention``), with the same ``scale``,
    ``soft_cap``, ``causal`` and ``sliding_window``.  Query row ``i`` is at position
    ``query_start + i`` (an int, or int32 [B]): ``causal`` keeps keys at or before it,
    ``sliding_window`` W those up to W before it.  With ``lengths`` (int32 [B]) keys
    from ``lengths[b]`` on are left out.  A row with ``lse`` -inf gives no weight.

    ``into`` (fp32 [B, Hkv, Skv], contiguous, apart from the inputs): the sums are added
    to it in place, and it is returned; otherwise a new tensor, 0 for keys left out.
    Deterministic.
    """
    return _lib.native().weight_sums(query, key, lse, causal, query_start, lengths, sliding_window, scale, soft_cap, into)


def evict_cache(key_cache, value_cache, scores, lengths, keep, recent=0, sinks=0, out=None):
    """Cut each sequence's cache to at most ``keep`` rows; returns ``(key, value,
    scores, slots, lengths)`` of the smaller cache.

    ``scores`` fp32 [B, Hkv, C]: the weight each row has accumulated
    (:func:`attention_weight_sums`).  Of a sequence with more than ``keep`` rows each
    KV head keeps the first ``sinks``, the last ``recent`` and those of the others
    with the largest scores (of equal ones the first; NaN counts as the largest), in
    their order; a shorter one stays whole.  ``slots`` int32 [B, Hkv, keep]: the old
    row of each new one, -1 behind the last; ``lengths`` int32 [B]: the new lengths.

    The new cache has ``keep`` rows, zero behind the last kept one; or ``out=(key,
    value, scores)`` receives it, tensors of one and the same number of rows (at least
    ``keep``, so that the cache can grow again) that share no memory with the old
    cache or each other.  Rows of ``out``'s key and value behind the last kept one are
    left as they were; its scores (contiguous fp32) are 0 there.  Lengths outside [0, C] count as
    the nearer end.
    """
    key, value, kept = (None, None, None) if out is None else out
    if out is not None and key is None:
        raise RuntimeError("out must be (key, value, scores)")
    return _lib.native().evict(key_cache, value_cache, scores, lengths, keep, recent, sinks, key, value, kept)
