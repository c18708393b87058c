"""Serving over a K/V cache on gfx950: new tokens into the cache, attention of a
tree of drafted tokens over it, the attention weight its keys have received, and
eviction by that weight.  No counterpart in the reference, which keeps no cache.

A cache is a pair of [B, Hkv, C, D] tensors (any strides a kernel can read in
place: innermost stride 1, rows on 16-byte boundaries) with ``lengths``, int32 [B]
on the device: the rows of each sequence that are in use.  ``lengths`` stays on the
device, so every call can be captured into a graph and replayed as the cache grows.

  rotary_append(...)          query' and the cache rows of new tokens, in one kernel
  tree_attention(...)         drafted tokens (or one new token) over cache and tree
  attention_weight_sums(...)  sum over the query rows of the softmax weights, per key
  evict_cache(...)            the rows worth keeping, copied to a smaller cache

None of them is differentiable.
"""
from __future__ import annotations

import math

import torch

import flexatt_lib as _lib
import flexatt_rotary as _rot
import npu_flash_attention as _nfa

__all__ = ["rotary_append", "tree_attention", "attention_weight_sums", "evict_cache"]


def _check_tensors(name_tensors, dtype, device):
    _nfa._check_device_dtype(name_tensors, dtype)
    grad = torch.is_grad_enabled()
    for name, t in name_tensors:
        if t.dim() != 4:
            raise RuntimeError(f"{name} must have four dimensions, got {tuple(t.shape)}")
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device} (got {t.device})")
        if grad and t.requires_grad:
            raise RuntimeError(f"{name} requires a gradient, which the cache operators do not have: "
                               "call them under torch.no_grad()")
    if dtype not in _nfa._DTYPES:
        raise RuntimeError(f"unsupported dtype {dtype} (expected float32, float16 or bfloat16)")
    D = name_tensors[0][1].shape[-1]
    if D not in _nfa._HEAD_DIMS:
        raise RuntimeError(f"unsupported head dim {D} (expected one of {_nfa._HEAD_DIMS})")


def _per_sequence(name, t, B, device):
    """An int32 [B] tensor of the call's device, contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (B,):
        raise RuntimeError(f"{name} must be an int32 tensor [B] = [{B}]")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device} (got {t.device})")
    return t if t.is_contiguous() else t.contiguous()


def _check_cache(query, key_cache, value_cache):
    B, Hq, _, D = query.shape
    assert key_cache.shape == value_cache.shape, "key and value cache shapes must match"
    assert key_cache.shape[0] == B, "query and cache batch sizes must match"
    assert key_cache.shape[3] == D, "query and cache head dims must match"
    assert key_cache.shape[1] > 0 and Hq % key_cache.shape[1] == 0, "Hq must be divisible by Hkv"


def _in_place(name, t):
    if not _nfa._kernel_ready(t):
        raise RuntimeError(f"{name} is written in place: its innermost stride must be 1 and its rows must start on "
                           "16-byte boundaries")
    return t


def _score_params(scale, soft_cap, sliding_window, D):
    """As the attention entry points: primitives are enabled by positive values."""
    return (float(scale) if scale is not None else 1.0 / math.sqrt(D),
            float(soft_cap) if soft_cap and soft_cap > 0.0 else 0.0,
            min(int(sliding_window), 0x7fffffff) if sliding_window and sliding_window > 0 else 0)


def rotary_append(query, key, value, key_cache, value_cache, lengths, inv_freq, positions=None, interleaved=False,
                  magnitude=1.0):
    """Put new tokens into the cache; returns ``query'``.

    ``query`` [B, Hq, S, D], ``key`` / ``value`` [B, Hkv, S, D]: the tokens behind the
    cached ones.  Rows ``lengths[b] + s`` of ``key_cache`` / ``value_cache`` receive the
    rotated key and the value of token ``s``, and ``query'`` is the rotated query, as
    :func:`flexatt_rotary.rotary_embedding` gives them; ``positions`` (int32 or int64
    [S] or [B, S]) defaults to the rows' numbers.  ``inv_freq=None`` rotates nothing
    and returns a copy of the query.  A row outside the cache is not written.
    ``lengths`` is read, not changed.
    """
    if not isinstance(query, torch.Tensor):
        raise RuntimeError("query must be a torch.Tensor")
    _check_tensors((("query", query), ("key", key), ("value", value), ("key_cache", key_cache),
                    ("value_cache", value_cache)), query.dtype, query.device)
    _check_cache(query, key_cache, value_cache)
    B, Hq, S, D = query.shape
    Hkv, C = key_cache.shape[1], key_cache.shape[2]
    assert key.shape == value.shape == (B, Hkv, S, D), "key and value must be [B, Hkv, S, D]"
    lengths = _per_sequence("lengths", lengths, B, query.device)
    if inv_freq is not None:
        inv_freq = _rot._check_frequencies(inv_freq, D, query.device)
    r = _rot._rotary_struct(query, Hkv, inv_freq, positions, interleaved, float(magnitude))
    qo = _rot._out_like(query)
    _in_place("key_cache", key_cache)
    _in_place("value_cache", value_cache)
    if C == 0:
        raise RuntimeError("the cache has no rows")
    if query.numel() == 0:
        return qo
    q, k, v = _nfa._prepare(query), _nfa._prepare(key), _nfa._prepare(value)
    with _nfa._device_guard(query.device):
        st = _lib.load().flexatt_rotary_append(r, _lib.tensor(q), _lib.tensor(k), _lib.tensor(v), _lib.tensor(qo),
                                               _lib.tensor(key_cache), _lib.tensor(value_cache), C, lengths.data_ptr(),
                                               _nfa._stream(query.device))
    _lib.check(st, "flexatt_rotary_append")
    return qo


def _tree_mask(tree_mask, B, T, device):
    """A tree mask in any accepted form as contiguous bytes [1 or B, T, T]."""
    m = tree_mask
    if not isinstance(m, torch.Tensor) or m.dtype.is_floating_point or m.dtype.is_complex:
        raise RuntimeError("tree_mask must be a bool or integer tensor")
    if m.dim() == 2:
        m = m.unsqueeze(0)
    if m.dim() != 3 or m.shape[0] not in (1, B) or m.shape[1] != T or m.shape[2] != T:
        raise RuntimeError(f"tree_mask must be [T, T] or [B, T, T] with B={B} and T={T}, got {tuple(tree_mask.shape)}")
    if m.device != device:
        raise RuntimeError(f"tree_mask must be on {device} (got {m.device})")
    m = m.view(torch.uint8) if m.dtype == torch.bool else m if m.dtype == torch.uint8 else (m != 0).view(torch.uint8)
    return m if m.is_contiguous() else m.contiguous()


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
    not read.

    ``sliding_window`` W keeps cached token ``j`` for drafted token ``t`` where
    ``lengths[b] + depths[b][t] - j <= W``; ``depths`` (int32 [T] or [B, T], 0 for a
    token directly behind the cached ones) defaults to ``t`` for a chain and must be
    given with a mask.  Within the tree the mask alone decides.  ``scale`` and
    ``soft_cap`` as in ``npu_flash_attention_forward``, and so are ``O`` (in
    ``query``'s dtype and layout), ``LSE`` (fp32 [B, Hq, T], natural log) and a token
    without keys (0 and -inf).  A sequence whose ``lengths[b] + T`` rows do not fit the
    cache, which only the device knows, gets NaN.
    """
    if not isinstance(query, torch.Tensor):
        raise RuntimeError("query must be a torch.Tensor")
    _check_tensors((("query", query), ("key_cache", key_cache), ("value_cache", value_cache)), query.dtype,
                   query.device)
    _check_cache(query, key_cache, value_cache)
    B, Hq, T, D = query.shape
    Hkv, C = key_cache.shape[1], key_cache.shape[2]
    if T > C:
        raise RuntimeError(f"{T} drafted tokens do not fit a cache of {C} rows")
    device = query.device
    lengths = _per_sequence("lengths", lengths, B, device)
    scale, soft_cap, window = _score_params(scale, soft_cap, sliding_window, D)
    p = _lib.Tree(_nfa._DTYPES[query.dtype], B, Hq, Hkv, T, C, D, scale, soft_cap, window)
    p.lengths = lengths.data_ptr()
    if tree_mask is not None:
        tree_mask = _tree_mask(tree_mask, B, T, device)
        p.mask_batch = tree_mask.shape[0]
        p.tree_mask = tree_mask.data_ptr()
    if window > 0:
        if depths is None and tree_mask is not None:
            raise RuntimeError("sliding_window with a tree_mask needs depths")
        if depths is not None:
            if not isinstance(depths, torch.Tensor) or depths.dtype != torch.int32 or depths.device != device:
                raise RuntimeError(f"depths must be an int32 tensor on {device}")
            if tuple(depths.shape) not in ((T,), (1, T), (B, T)):
                raise RuntimeError(f"depths must be [T] or [B, T] = [{B}, {T}], got {tuple(depths.shape)}")
            depths = depths.expand(B, T).contiguous()
            p.depths = depths.data_ptr()
    O = _rot._out_like(query)
    LSE = torch.empty(B, Hq, T, device=device, dtype=torch.float32)
    if query.numel() == 0:
        return (O, LSE) if return_lse else O
    lib = _lib.load()
    q, k, v = _nfa._prepare(query), _nfa._prepare(key_cache), _nfa._prepare(value_cache)
    with _nfa._device_guard(device):
        n = lib.flexatt_tree_fwd_workspace(p)
        ws = torch.empty(n, dtype=torch.uint8, device=device) if 0 < n < 1 << 62 else None
        st = lib.flexatt_tree_fwd(p, _lib.tensor(q), _lib.tensor(k), _lib.tensor(v), _lib.tensor(O), LSE.data_ptr(),
                                  None if ws is None else ws.data_ptr(), 0 if ws is None else n, _nfa._stream(device))
    _lib.check(st, "flexatt_tree_fwd")
    return (O, LSE) if return_lse else O


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

    ``into`` (fp32 [B, Hkv, Skv], contiguous): the sums are added to it in place, and
    it is returned; otherwise a new tensor, 0 for keys left out.  Deterministic.
    """
    if not isinstance(query, torch.Tensor):
        raise RuntimeError("query must be a torch.Tensor")
    device = query.device
    _check_tensors((("query", query), ("key", key)), query.dtype, device)
    B, Hq, Sq, D = query.shape
    Hkv, Sk = key.shape[1], key.shape[2]
    assert key.shape[0] == B, "query and key batch sizes must match"
    assert key.shape[3] == D, "query and key head dims must match"
    assert Hkv > 0 and Hq % Hkv == 0, "Hq must be divisible by Hkv"
    assert isinstance(lse, torch.Tensor) and tuple(lse.shape) == (B, Hq, Sq), "lse must be [B, Hq, Sq]"
    if lse.device != device:
        raise RuntimeError(f"lse must be on {device} (got {lse.device})")
    if lse.dtype != torch.float32 or not lse.is_contiguous():
        lse = lse.to(torch.float32).contiguous()
    scale, soft_cap, window = _score_params(scale, soft_cap, sliding_window, D)
    p = _lib.Weights(_nfa._DTYPES[query.dtype], B, Hq, Hkv, Sq, Sk, D, scale, soft_cap, 1 if causal else 0, window)
    if isinstance(query_start, torch.Tensor):
        query_start = _per_sequence("query_start", query_start, B, device)
        p.query_starts = query_start.data_ptr()
    else:
        if not -(1 << 31) <= int(query_start) < 1 << 31:
            raise RuntimeError("query_start must fit 32 bits")
        p.query_start = int(query_start)
    if lengths is not None:
        lengths = _per_sequence("lengths", lengths, B, device)
        p.lengths = lengths.data_ptr()
    if into is not None:
        if not isinstance(into, torch.Tensor) or into.dtype != torch.float32 or tuple(into.shape) != (B, Hkv, Sk) \
                or into.device != device or not into.is_contiguous():
            raise RuntimeError(f"into must be a contiguous fp32 [B, Hkv, Skv] = [{B}, {Hkv}, {Sk}] tensor on {device}")
        p.accumulate = 1
    sums = into if into is not None else torch.empty(B, Hkv, Sk, dtype=torch.float32, device=device)
    if sums.numel() == 0:
        return sums
    if query.numel() == 0:
        return sums if into is not None else sums.zero_()
    lib = _lib.load()
    q, k = _nfa._prepare(query), _nfa._prepare(key)
    with _nfa._device_guard(device):
        n = lib.flexatt_weight_sums_workspace(p)
        ws = torch.empty(n, dtype=torch.uint8, device=device) if 0 < n < 1 << 62 else None
        st = lib.flexatt_weight_sums(p, _lib.tensor(q), _lib.tensor(k), lse.data_ptr(), sums.data_ptr(),
                                     None if ws is None else ws.data_ptr(), 0 if ws is None else n,
                                     _nfa._stream(device))
    _lib.check(st, "flexatt_weight_sums")
    return sums


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
    cache.  Rows of ``out``'s key and value behind the last kept one are left as they
    were; its scores (contiguous fp32) are 0 there.  Lengths outside [0, C] count as
    the nearer end.
    """
    if not isinstance(key_cache, torch.Tensor):
        raise RuntimeError("key_cache must be a torch.Tensor")
    device = key_cache.device
    _check_tensors((("key_cache", key_cache), ("value_cache", value_cache)), key_cache.dtype, device)
    assert key_cache.shape == value_cache.shape, "key and value cache shapes must match"
    B, H, C, D = key_cache.shape
    if key_cache.numel() == 0:
        raise RuntimeError("the cache has no rows")
    if not isinstance(scores, torch.Tensor) or scores.dtype != torch.float32 or tuple(scores.shape) != (B, H, C) \
            or scores.device != device:
        raise RuntimeError(f"scores must be an fp32 [B, Hkv, C] = [{B}, {H}, {C}] tensor on {device}")
    scores = scores if scores.is_contiguous() else scores.contiguous()
    lengths = _per_sequence("lengths", lengths, B, device)
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if keep < 1 or keep >= 1 << 31 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise RuntimeError("keep must be at least 1, recent and sinks at least 0 and together at most keep")
    if out is None:
        ko = torch.empty(B, H, keep, D, dtype=key_cache.dtype, device=device)
        vo = torch.empty(B, H, keep, D, dtype=key_cache.dtype, device=device)
        so = torch.empty(B, H, keep, dtype=torch.float32, device=device)
    else:
        ko, vo, so = out
        _check_tensors((("out key", ko), ("out value", vo)), key_cache.dtype, device)
        rows = ko.shape[2]
        if tuple(ko.shape) != (B, H, rows, D) or ko.shape != vo.shape or rows < keep:
            raise RuntimeError(f"out key and value must be [B, Hkv, at least keep, D] = [{B}, {H}, {keep}, {D}]")
        _in_place("out key", ko)
        _in_place("out value", vo)
        if not isinstance(so, torch.Tensor) or so.dtype != torch.float32 or tuple(so.shape) != (B, H, rows) \
                or so.device != device or not so.is_contiguous():
            raise RuntimeError(f"out scores must be a contiguous fp32 [{B}, {H}, {rows}] tensor on {device}")
    slots = torch.empty(B, H, keep, dtype=torch.int32, device=device)
    new_lengths = torch.empty(B, dtype=torch.int32, device=device)
    p = _lib.Evict(_nfa._DTYPES[key_cache.dtype], B, H, C, D, keep, recent, sinks, ko.shape[2],
                   1 if out is None else 0)
    p.lengths = lengths.data_ptr()
    k, v = _nfa._prepare(key_cache), _nfa._prepare(value_cache)
    with _nfa._device_guard(device):
        st = _lib.load().flexatt_evict_rows(p, _lib.tensor(k), _lib.tensor(v), scores.data_ptr(), _lib.tensor(ko),
                                            _lib.tensor(vo), so.data_ptr(), slots.data_ptr(), new_lengths.data_ptr(),
                                            _nfa._stream(device))
    _lib.check(st, "flexatt_evict_rows")
    return ko, vo, so, slots, new_lengths
