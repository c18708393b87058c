"""float64 CPU oracle of the cache operators and rotary positions (test infrastructure only).

Plain loops over sequences and heads, written from the operators' definitions.  Beside each result stand the bounds
that the kernels' arithmetic has to keep, so that the tests' tolerances follow from the inputs.
"""
import math

import torch

EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def rotary(x, inv_freq, positions, interleaved=False, magnitude=1.0, inverse=False):
    """x [B, H, S, D] (float64), positions [B, S]: the rotation, and how far a kernel may be off per element.

    The kernel's sine and cosine are off by less than 2^-22 (argument 2^-24, series 2^-25, three roundings), the two
    products and the sum round at 2^-24 each: 2^-21 m (|x1| + |x2|) in all, and one rounding to the type."""
    r2 = inv_freq.numel()
    y, slack = x.clone(), torch.zeros_like(x)
    ang = positions.double()[:, None, :, None] * inv_freq.double() * (-1.0 if inverse else 1.0)
    c, s = ang.cos() * magnitude, ang.sin() * magnitude
    first, second = (slice(0, 2 * r2, 2), slice(1, 2 * r2, 2)) if interleaved else (slice(0, r2), slice(r2, 2 * r2))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    slack[..., first] = slack[..., second] = 2.0 ** -21 * abs(magnitude) * (a.abs() + b.abs())
    return y, slack


def rounded(y, slack, dtype):
    """The tolerance of y rounded to dtype, half a step (the smallest numbers have an absolute step)."""
    eps = EPS[dtype]
    return slack + (y.abs() + slack) * eps / 2 + torch.finfo(dtype).tiny * eps


def tree_allowed(n, T, C, mask, window, depths):
    """[T, C] bool: the cache rows each drafted token of one sequence of n cached tokens sees."""
    ok = torch.zeros(T, C, dtype=torch.bool)
    for t in range(T):
        lo = 0 if not window else max(0, n + (t if depths is None else max(int(depths[t]), 0)) - window)
        ok[t, lo:n] = True
        ok[t, n:n + T] = (torch.arange(T) <= t) if mask is None else mask[t] != 0
    return ok


def _scores(q, k, scale, cap):
    """Scores of one (sequence, KV head) and a bound of the kernel's error of each: products of the inputs are exact
    in fp32 (or rounded at 2^-24), sums of D terms round at (D + 4) 2^-24 of the sum of magnitudes, the soft-cap's
    exponential and reciprocal at cap 2^-21, log2 units and the difference to the maximum or LSE at 2^-22 |x|."""
    x = q @ k.transpose(-1, -2) * scale
    err = (q.abs() @ k.abs().transpose(-1, -2)) * (abs(scale) * (q.shape[-1] + 4) * 2.0 ** -24)
    if cap:
        x = cap * torch.tanh(x / cap)
        err = err + cap * 2.0 ** -21
    return x, err + x.abs() * 2.0 ** -22


def tree_attention(q, kc, vc, lengths, mask=None, window=0, depths=None, scale=None, cap=0.0, dtype=torch.bfloat16):
    """O, LSE and their tolerances; mask [T, T] or [B, T, T], depths [B, T] or None.

    P is rounded to the type before P V (fp32: not at all): half a step of each weight, and for fp16, whose weights
    under 2^-14 have the step 2^-24, n 2^-25 in all beside a largest weight of at least 1.  A score error e scales a
    weight by exp(e) and so the row sum: 2 e max|v|."""
    B, Hq, T, D = q.shape
    Hkv, C = kc.shape[1:3]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    O = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    LSE = torch.full((B, Hq, T), float("-inf"), dtype=torch.float64)
    tO, tL = torch.zeros_like(O), torch.zeros_like(LSE)
    half = 0.0 if dtype == torch.float32 else EPS[dtype] / 2
    for b in range(B):
        n = int(lengths[b])
        if n < 0 or n + T > C:
            O[b], LSE[b] = float("nan"), float("nan")
            continue
        m = None if mask is None else mask[b % mask.shape[0]] if mask.dim() == 3 else mask
        ok = tree_allowed(n, T, C, m, window, None if depths is None else depths[b])[:, :n + T]
        for h in range(Hq):
            k, v = kc[b, h // G, :n + T].double(), vc[b, h // G, :n + T].double()
            x, e = _scores(q[b, h].double(), k, scale, cap)
            x = x.masked_fill(~ok, float("-inf"))
            lse = torch.logsumexp(x, dim=-1)
            some = ok.any(dim=-1)
            p = torch.exp(x - torch.where(some, lse, torch.zeros_like(lse))[:, None])
            o = p @ v
            e = e.masked_fill(~ok, 0.0).amax(dim=-1)
            vmax = torch.where(ok[:, :, None], v.abs()[None], torch.zeros(())).amax(dim=(1, 2))
            O[b, h] = o
            LSE[b, h] = lse
            flat = (n + T) * 2.0 ** -25 if dtype == torch.float16 else 0.0
            loose = ((half + 2 * e + flat + 2.0 ** -20) * vmax)[:, None].expand_as(o)
            tO[b, h] = rounded(o, loose, dtype)
            tL[b, h] = e + torch.where(some, lse.abs(), torch.zeros_like(lse)) * 2.0 ** -21 + 2.0 ** -20
    return O, LSE, tO, tL


def weight_sums(q, k, lse, causal=False, starts=None, lengths=None, window=0, scale=None, cap=0.0):
    """Sums and their tolerances.  A weight is off by its score's error and by LSE's rounding at 2^-22 |LSE|; a sum of
    R = G Sq rows rounds at (R + 8) 2^-24 of itself at most."""
    B, Hq, Sq, D = q.shape
    Hkv, C = k.shape[1:3]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    w = torch.zeros(B, Hkv, C, dtype=torch.float64)
    tol = torch.zeros_like(w)
    for b in range(B):
        n = C if lengths is None else min(max(int(lengths[b]), 0), C)
        s0 = 0 if starts is None else int(starts[b]) if torch.is_tensor(starts) else starts
        i, j = torch.arange(Sq)[:, None] + s0, torch.arange(n)[None, :]
        ok = torch.ones(Sq, n, dtype=torch.bool)
        if causal:
            ok &= j <= i
        if window:
            ok &= i - j <= window
        for h in range(Hq):
            x, e = _scores(q[b, h].double(), k[b, h // G, :n].double(), scale, cap)
            row = lse[b, h].double()[:, None]
            p = torch.where(ok & (row != float("-inf")), torch.exp(x - row), torch.zeros(()).double())
            w[b, h // G, :n] += p.sum(dim=0)
            tol[b, h // G, :n] += (p * (2 * e + row.abs().nan_to_num(posinf=0.0) * 2.0 ** -22 + 2.0 ** -21)).sum(dim=0)
    return w, tol + w * (G * Sq + 8) * 2.0 ** -24 + 2.0 ** -100


def evict(scores, n, keep, recent, sinks):
    """The kept slots of one (sequence, head): a list in order.  scores: floats, NaN the largest."""
    if n <= keep:
        return list(range(n))
    free = range(sinks, n - recent)
    rank = sorted(free, key=lambda j: (0 if math.isnan(scores[j]) else 1, 0.0 if math.isnan(scores[j]) else -scores[j], j))
    return sorted(list(range(sinks)) + list(range(n - recent, n)) + rank[:keep - sinks - recent])
