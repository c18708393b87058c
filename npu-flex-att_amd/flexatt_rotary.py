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


def rotary_embedding(query, key, inv_freq, positions=None, interleaved=False, magnitude=1.0):
    """Rotary positions: ``(query', key')``, each in its input's dtype and layout.

    ``query`` [B, Hq, S, D] and ``key`` [B, Hkv, S, D] (or None, then ``key'`` is
    None); any strides.  The first ``2 * len(inv_freq)`` elements of each head are
    turned, the rest is copied.  Pair ``i`` is elements ``(i, i + len(inv_freq))``, or
    ``(2 i, 2 i + 1)`` with ``interleaved``; its angle is ``positions * inv_freq[i]``,
    formed in 64 bits, and ``magnitude`` scales both of its elements (see
    :func:`rotary_frequencies`).  ``positions``: int32 or int64 [S] or [B, S];
    default 0, 1, ....

    Differentiable in query and key, in reverse mode; an argument that carries a tangent
    is refused, and so is, with gradients on, an ``inv_freq`` that requires them.  A
    backward pass may be captured into a graph, as any of torch's, while no eager graph
    of the same leaves is alive.  Small calls wait for autograd's hand-over to its device
    thread; inside ``torch.autograd.set_multithreading_enabled(False)`` there is none.
    Not traceable (``make_fx``, export, fake tensors); ``torch.compile`` breaks its graph
    here.
    """
    return _lib.native().rotary(query, key, inv_freq, positions, interleaved, magnitude)
