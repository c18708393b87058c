"""Rotary positions for the queries and keys of an attention call, on gfx950.

The reference has no positional embedding beside ALiBi: its callers hand over
queries and keys that are already positioned.  These entry points do that step
with one HIP kernel (``flexatt_rotary_apply`` in include/flexatt.h) in front of
``npu_flex_attention`` and its relatives; :mod:`flexatt_cache` holds the form that
also writes new tokens into a K/V cache.

  rotary_frequencies(...)  angles per position of each pair, scaled for long contexts
  rotary_embedding(...)    differentiable rotation of query and key
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

import flexatt_lib as _lib
import npu_flash_attention as _nfa

__all__ = ["rotary_frequencies", "rotary_embedding"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 0, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, magnitude)`` for :func:`rotary_embedding`: the angle of one
    position for each of the ``rotary_dim / 2`` pairs, in 64 bits, and the factor
    that goes with it.

    ``scaling`` extends a context of ``original_length`` by ``factor``:

    * ``None``: ``base ** (-2 i / rotary_dim)``;
    * ``"linear"``: all of them divided by ``factor``;
    * ``"ntk"``: the base raised so that the slowest pair is divided by ``factor``;
    * ``"turns"``: pairs that make at most ``slow`` turns over the original length are
      divided by ``factor``, those that make ``fast`` or more stay, and the share of
      each runs linearly with the turns between them;
    * ``"yarn"``: the same with the share linear in the pair's index between the
      (rounded) indices of those two pairs, and a magnitude of ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in (None, "linear", "ntk", "turns", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling is not None and not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling in ("turns", "yarn") and not (original_length > 0 and fast > slow > 0.0):
        raise ValueError(f"{scaling} scaling needs original_length > 0 and fast > slow > 0")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = torch.as_tensor(base, dtype=torch.float64) ** (-i / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("turns", "yarn"):
        if scaling == "turns":
            kept = (original_length * freq / (2.0 * math.pi) - slow) / (fast - slow)
        else:
            def index(turns):  # the pair that makes so many turns over the original length
                return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

            first = max(math.floor(index(fast)), 0)
            last = min(math.ceil(index(slow)), rotary_dim - 1)
            kept = 1.0 - (i / 2 - first) / max(last - first, 0.001)
            magnitude = 0.1 * math.log(factor) + 1.0
        kept = kept.clamp(0.0, 1.0)
        freq = freq * kept + freq / factor * (1.0 - kept)
    return freq.to(device), magnitude


def _check_frequencies(inv_freq, D, device):
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1:
        raise RuntimeError("inv_freq must be a float64 tensor with one entry per pair (see rotary_frequencies)")
    if inv_freq.device != device:
        raise RuntimeError(f"inv_freq must be on {device} (got {inv_freq.device})")
    if 2 * inv_freq.numel() > D:
        raise RuntimeError(f"inv_freq has {inv_freq.numel()} pairs, a head of {D} elements has {D // 2}")
    return inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous()


def _check_positions(positions, B, S, device):
    """Positions as int32 or int64 [S] or [B|1, S]: the tensor and its strides."""
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("positions must be an int32 or int64 tensor")
    if positions.device != device:
        raise RuntimeError(f"positions must be on {device} (got {positions.device})")
    if positions.dim() == 1 and positions.shape[0] == S:
        return 0, positions.stride(0)
    if positions.dim() == 2 and positions.shape[1] == S and positions.shape[0] in (1, B):
        return positions.stride(0) if positions.shape[0] > 1 else 0, positions.stride(1)
    raise RuntimeError(f"positions must be [S] or [B, S] = [{B}, {S}], got {tuple(positions.shape)}")


def _rotary_struct(query, Hkv, inv_freq, positions, interleaved, magnitude, inverse=False):
    """The C description of a rotation of ``query``'s tokens (``inv_freq`` already
    checked, or None: nothing is turned)."""
    B, Hq, S, D = query.shape
    if D not in _nfa._HEAD_DIMS:
        raise RuntimeError(f"unsupported head dim {D} (expected one of {_nfa._HEAD_DIMS})")
    if query.dtype not in _nfa._DTYPES:
        raise RuntimeError(f"unsupported dtype {query.dtype} (expected float32, float16 or bfloat16)")
    r = _lib.Rotary(_nfa._DTYPES[query.dtype], B, Hq, Hkv, S, D, 0, 1 if interleaved else 0, 1 if inverse else 0,
                    magnitude)
    if inv_freq is not None and inv_freq.numel() > 0:
        r.rotary_dim = 2 * inv_freq.numel()
        r.inv_freq = inv_freq.data_ptr()
    if positions is not None:
        r.position_stride_b, r.position_stride_s = _check_positions(positions, B, S, query.device)
        r.positions = positions.data_ptr()
        r.position_bytes = positions.element_size()
    return r


def _out_like(t):
    o = torch.empty_like(t)
    if not o.is_contiguous() and not _nfa._kernel_ready(o):
        o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return o


def _rotate(query, key, inv_freq, positions, interleaved, magnitude, inverse):
    """The kernel call: (query', key') or (query', None)."""
    inv_freq = _check_frequencies(inv_freq, query.shape[-1], query.device)
    r = _rotary_struct(query, 0 if key is None else key.shape[1], inv_freq, positions, interleaved, magnitude, inverse)
    qo, ko = _out_like(query), None if key is None else _out_like(key)
    if query.numel() == 0 and (key is None or key.numel() == 0):
        return qo, ko
    q = _nfa._prepare(query)
    k = None if key is None else _nfa._prepare(key)
    with _nfa._device_guard(query.device):
        st = _lib.load().flexatt_rotary_apply(r, _lib.tensor(q), None if k is None else _lib.tensor(k),
                                              _lib.tensor(qo), None if ko is None else _lib.tensor(ko),
                                              _nfa._stream(query.device))
    _lib.check(st, "flexatt_rotary_apply")
    return qo, ko


class _Rotary(torch.autograd.Function):
    """The rotation is linear, and its transpose turns the other way: the backward
    pass is this function again (so gradients of gradients work too)."""

    @staticmethod
    def forward(ctx, query, key, inv_freq, positions, interleaved, magnitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(inv_freq, positions)
        ctx.how = (interleaved, magnitude, inverse)
        qo, ko = _rotate(query, key, inv_freq, positions, interleaved, magnitude, inverse)
        return qo if key is None else (qo, ko)

    @staticmethod
    def backward(ctx, dq, dk=None):
        inv_freq, positions = ctx.saved_tensors
        interleaved, magnitude, inverse = ctx.how
        how = (inv_freq, positions, interleaved, magnitude, not inverse)
        if dq is not None and dk is not None:
            dq, dk = _Rotary.apply(dq, dk, *how)
        elif dq is not None:
            dq = _Rotary.apply(dq, None, *how)
        elif dk is not None:
            dk = _Rotary.apply(dk, None, *how)
        return dq, dk, None, None, None, None, None


def rotary_embedding(query, key, inv_freq, positions=None, interleaved=False, magnitude=1.0):
    """Rotary positions: ``(query', key')``, each in its input's dtype and layout.

    ``query`` [B, Hq, S, D] and ``key`` [B, Hkv, S, D] (or None, then ``key'`` is
    None); any strides.  The first ``2 * len(inv_freq)`` elements of each head are
    turned, the rest is copied.  Pair ``i`` is elements ``(i, i + len(inv_freq))``, or
    ``(2 i, 2 i + 1)`` with ``interleaved``; its angle is ``positions * inv_freq[i]``,
    formed in 64 bits, and ``magnitude`` scales both of its elements (see
    :func:`rotary_frequencies`).  ``positions``: int32 or int64 [S] or [B, S];
    default 0, 1, ....  Differentiable in query and key.
    """
    if not isinstance(query, torch.Tensor) or query.dim() != 4:
        raise RuntimeError("query must be a [B, Hq, S, D] tensor")
    _nfa._check_device_dtype((("query", query),) if key is None else (("query", query), ("key", key)), query.dtype)
    if key is not None:
        assert key.dim() == 4 and key.shape[0] == query.shape[0] and key.shape[2:] == query.shape[2:], \
            "query and key must have the same batch, length and head dim"
        if key.device != query.device:
            raise RuntimeError(f"key must be on {query.device} (got {key.device})")
    magnitude = float(magnitude)
    if not math.isfinite(magnitude):
        raise RuntimeError("magnitude must be finite")
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)):
        out = _Rotary.apply(query, key, inv_freq, positions, bool(interleaved), magnitude, False)
        return (out, None) if key is None else out
    return _rotate(query, key, inv_freq, positions, interleaved, magnitude, False)
