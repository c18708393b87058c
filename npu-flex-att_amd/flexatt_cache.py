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
  norm_rotary_append(...)     rotary_append behind a norm of each head of query and key
  shared_prefix_attention(...)  tree_attention behind a prefix that all sequences share

A cache may hold 8 bits an element: ``key_cache`` / ``value_cache`` of float8_e4m3fn or
int8 and ``key_scales`` / ``value_scales``, float32 [B, Hkv, C] (contiguous where they
are written), one scale for each row of each head; a row stands for codes * scale.

  quantized_append(...)          the appends, into such a cache
  dequantize_cache(...)          such a cache in a wider type again
  quantized_tree_attention(...)  tree_attention over such a cache

None of them is differentiable: a tensor that carries a tangent, or with gradients
on one that requires them, is refused.  Nor can they be traced (``make_fx``, export,
fake tensors); ``torch.compile`` breaks its graph at them.
"""
from __future__ import annotations

import torch

import flexatt_lib as _lib

__all__ = ["rotary_append", "tree_attention", "attention_weight_sums", "evict_cache", "norm_rotary_append",
           "shared_prefix_attention", "quantized_append", "dequantize_cache", "quantized_tree_attention"]


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


def norm_rotary_append(query, key, value, key_cache, value_cache, lengths, query_weight, key_weight, inv_freq,
                       positions=None, interleaved=False, magnitude=1.0, eps=1e-6):
    """:func:`rotary_append` with each head of query and key normalised before its rotation,
    as :func:`flexatt_rotary.norm_rotary_embedding` does it.  ``inv_freq=None`` rotates
    nothing.
    """
    return _lib.native().norm_rotary_append(query, key, value, key_cache, value_cache, lengths, query_weight, key_weight,
                                            inv_freq, positions, interleaved, magnitude, eps)


def shared_prefix_attention(query, prefix_key, prefix_value, key_cache, value_cache, lengths, tree_mask=None,
                            sliding_window=0, depths=None, scale=None, soft_cap=0.0, return_lse=False):
    """:func:`tree_attention` of sequences that share a prefix, whose keys are read once for
    all of them.

    ``prefix_key`` / ``prefix_value`` [Hkv, P, D], in the cache's dtype: the keys and values
    of the prefix's positions 0 .. P - 1, of which every drafted token sees all (for a
    shorter prefix in a larger buffer pass a slice).  Row ``j`` of a sequence's own cache is
    position ``P + j``: append to it with ``positions`` that say so.  The other arguments
    and results are those of :func:`tree_attention`; ``sliding_window`` W counts positions,
    so it keeps row ``j`` of the prefix where ``P + lengths[b] + depths[b][t] - j <= W``.

    Weights are rounded to the type for the second product, as there, but not where all
    sequences' query rows of a KV head (B, T and Hq / Hkv multiplied) are 32 or fewer, or with
    a head dim of 256: what the rounding leaves is added.
    """
    return _lib.native().prefix_attention(query, prefix_key, prefix_value, key_cache, value_cache, lengths, tree_mask,
                                          sliding_window, depths, scale, soft_cap, return_lse)


def quantized_append(query, key, value, key_cache, value_cache, key_scales, value_scales, lengths, inv_freq,
                     positions=None, interleaved=False, magnitude=1.0, query_weight=None, key_weight=None, eps=1e-6):
    """:func:`rotary_append`, with both weights :func:`norm_rotary_append`, into a cache of 8
    bits; returns ``query'``, in query's dtype.

    A row's scale is its largest size (at least 2 ** -100) over the largest code, 448
    (float8_e4m3fn) or 127 (int8), and its codes are the values over the scale, rounded to
    the nearest, of two the even one; keys are rounded nowhere before, and what decides a
    code is in 64 bits.  A row with an infinity or NaN, be it by a weight or a frequency, gets
    codes of 0 and a scale of NaN.
    Rows of the cache and its scales that no token goes to are left as they were; the new
    tokens, both caches and both scales share no memory.
    """
    return _lib.native().quant_append(query, key, value, key_cache, value_cache, key_scales, value_scales, lengths, inv_freq,
                                      positions, interleaved, magnitude, query_weight, key_weight, eps)


def dequantize_cache(key_cache, value_cache, key_scales, value_scales, lengths, dtype=torch.bfloat16, out=None):
    """``(key, value)`` [B, Hkv, C, D] of ``dtype`` (float32, float16, bfloat16): codes times
    scales, rounded once, of the first ``lengths[b]`` rows of each sequence (outside [0, C]
    the nearer end) and zeros behind them.

    ``out=(key, value)`` receives them instead, in its own dtype, tensors that share no
    memory with the cache or each other; rows behind the lengths are left as they were.
    """
    key, value = (None, None) if out is None else out
    if out is not None and (key is None or value is None):
        raise RuntimeError("out must be (key, value)")
    return _lib.native().dequant(key_cache, value_cache, key_scales, value_scales, lengths, dtype, key, value)


def quantized_tree_attention(query, key_cache, value_cache, key_scales, value_scales, lengths, tree_mask=None,
                             sliding_window=0, depths=None, scale=None, soft_cap=0.0, return_lse=False):
    """:func:`tree_attention` over a cache of 8 bits, for float16 and bfloat16 queries; the
    other arguments and results are the same.

    Scores are products with the codes times the key's scale, in 32 bits.  A weight times its
    value's scale is rounded to float16 (for float16 queries to two of them), in which the
    largest scale that the token sees is 2 ** 6 at least: a value 2 ** 20 times smaller than
    the largest keeps eleven bits of a weight of 1.  A ``tree_mask`` is of 2 ** 15 tokens at
    most.  Scales of rows that a token does not see may be anything, their codes anything but
    float8_e4m3fn's NaN.
    """
    return _lib.native().quant_tree_attention(query, key_cache, value_cache, key_scales, value_scales, lengths, tree_mask,
                                              sliding_window, depths, scale, soft_cap, return_lse)
