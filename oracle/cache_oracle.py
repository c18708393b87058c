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

    P is rounded to the type before P V (fp32: not at all): half a step of each weight, and for fp16, whose weights under
    2^-14 have the step 2^-24, 2^-25 of each value, over the row's sum of weights relative to a largest of at least 1.  A
    score error e scales a weight by exp(e) and so the row sum: 2 e; exponentials and partials are at 2^-20, and an
    accumulator rounds at most once for two keys (fp32: two products a time, of half the tiles; 16 bits: sixteen): (n + T) /
    2 + 16 roundings at 2^-24.  All but fp16's smallest step are shares of the sum of weights times |values|."""
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
            e = e.masked_fill(~ok, 0.0).amax(dim=-1)
            share = half + 2 * e + 2.0 ** -20 + ((n + T) / 2 + 16) * 2.0 ** -24
            loose = (p @ v.abs()) * share[:, None]
            if dtype == torch.float16:  # (p.amax: the largest weight over the row's sum)
                loose = loose + (ok.double() @ v.abs()) * p.amax(dim=-1, keepdim=True) * 2.0 ** -25
            O[b, h] = p @ v
            LSE[b, h] = lse
            tO[b, h] = rounded(O[b, h], loose, dtype)
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


def norm_rotary(x, w, inv_freq, positions, interleaved=False, magnitude=1.0, eps=1e-6):
    """x [B, H, S, D], w [D] (float64): each head normalised and turned, and how far a kernel may be off per element.

    A row's sum of squares has at most 16 fused steps a lane and 5 joins, 21 2^-24 of itself, the mean, eps and the
    reciprocal root three more: 2^-20 of r in all.  Weight times sine and the product with r round twice more than the
    rotation alone: 2^-19 (|x1 w1| + |x2 w2|) r."""
    r = 1.0 / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt()
    y, slack = rotary(x * r * w, inv_freq, positions, interleaved, magnitude)
    return y, slack * 4 + (x * r * w).abs() * 2.0 ** -19


def norm_rotary_grad(x, w, gy, inv_freq, positions, interleaved=False, magnitude=1.0, eps=1e-6):
    """The gradients of x and w, with their bounds: ((dx, slack), (dw, slack)).

    g, the gradient turned back, is off by the rotation's bound; r by 2^-20 of itself; the row's sum of g w x by 24 2^-24
    of its magnitudes.  dw adds up B S H products: a lane's heads one after the other, then at most 40 joins."""
    D = x.shape[-1]
    r = 1.0 / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt()
    g, eg = rotary(gy, inv_freq, positions, interleaved, magnitude, inverse=True)
    gw = g * w
    dot = (gw * x).sum(dim=-1, keepdim=True)
    dx = r * (gw - x * (r * r / D) * dot)
    off = (eg * (w * x).abs()).sum(dim=-1, keepdim=True) + (gw * x).abs().sum(dim=-1, keepdim=True) * 2.0 ** -18
    sx = r * (eg * w.abs() + gw.abs() * 2.0 ** -19 + x.abs() * (r * r / D) * off)
    terms = g * x * r
    dw = terms.sum(dim=(0, 1, 2))
    sw = (eg * (x * r).abs() + terms.abs() * (2.0 ** -19 + (x.shape[1] + 40) * 2.0 ** -24)).sum(dim=(0, 1, 2))
    return (dx, sx), (dw, sw)


TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def scale_of(y, code):
    """The scales of rows y [..., D] (float64)."""
    return y.abs().amax(dim=-1).clamp(min=2.0 ** -100) / TOP[code]


def code_tolerance(y, slack, scale, code):
    """How far code * scale may be from y, which the kernel has to `slack`: half a code's step (int8: half a scale; e4m3:
    2^-4 of the value, at least half of its smallest step 2^-9), 2^-22 of the value for the scale's and quotient's
    roundings."""
    half = scale[..., None] / 2 if code == torch.int8 else torch.maximum(y.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10)
    return half + slack * (1 + 2.0 ** -4) + y.abs() * 2.0 ** -21


def quantized_tree_attention(q, kc, vc, ks, vs, lengths, mask=None, window=0, depths=None, scale=None, cap=0.0,
                             dtype=torch.bfloat16):
    """O, LSE and their tolerances: those of :func:`tree_attention` over codes * scales, but for what the second product
    rounds.

    The scales add two roundings to a score, 2^-23 of it.  A weight's exponent is at most 64 in log2 units, rounded at
    2^-19, and the exponential, the scale and the partials at 2^-20 together.  The weight times its value's scale is rounded
    to fp16: 2^-11 of it, 2^-22 for fp16 queries, whose rest is a second operand.  It is held relative to the largest scale
    S that the row has met, S between 2^6 and 2^7, and to a largest weight of at least 2^-1/2, so half of fp16's smallest
    step, 2^-25, is S 2^-30.5 for a code of 1: (n + T) S top 2^-30.5 over the row's sum of weights, relative to the largest.
    An accumulator takes two MFMAs of sixteen products from every fourth 32-key tile: (n + T) / 4 + 16 roundings at 2^-24
    with the joins.  All but the smallest step's are shares of the sum of weights times |values|."""
    B, Hq, T, D = q.shape
    G, C, top = Hq // kc.shape[1], kc.shape[2], TOP[kc.dtype]
    seen = [0 <= int(n) <= C - T for n in lengths]
    k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    O, LSE, tO, tL = tree_attention(q, k, v, lengths, mask, window, depths, scale, cap, dtype)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        if not seen[b]:
            continue
        n = int(lengths[b])
        m = None if mask is None else mask[b % mask.shape[0]] if mask.dim() == 3 else mask
        ok = tree_allowed(n, T, C, m, window, None if depths is None else depths[b])[:, :n + T]
        for h in range(Hq):
            kk, vv, s = k[b, h // G, :n + T], v[b, h // G, :n + T], vs[b, h // G, :n + T].double()
            x, e = _scores(q[b, h].double(), kk, scale, cap)
            size = (q[b, h].double().abs() @ kk.abs().T * abs(scale)).masked_fill(~ok, 0.0).amax(dim=-1)
            e = e.masked_fill(~ok, 0.0).amax(dim=-1) + size * 2.0 ** -23
            x = x.masked_fill(~ok, float("-inf"))
            w = torch.exp(x - x.amax(dim=-1, keepdim=True)).nan_to_num(nan=0.0)
            row = w.sum(dim=-1).clamp(min=1.0)
            part = (w @ vv.abs()) / row[:, None]
            half = 2.0 ** -22 if dtype == torch.float16 else 2.0 ** -11
            share = half + 2 * e + 2.0 ** -19 + 2.0 ** -20 + ((n + T) / 4 + 16) * 2.0 ** -24
            largest = torch.where(ok, s[None], torch.zeros(())).amax(dim=-1)
            least = (n + T) * 2.0 ** -30.5 * largest * top / row
            tO[b, h] = rounded(O[b, h], part * share[:, None] + least[:, None], dtype)
            tL[b, h] += size * 2.0 ** -23 + 2.0 ** -19
    return O, LSE, tO, tL


def prefix_attention(q, pk, pv, kc, vc, lengths, mask=None, window=0, depths=None, scale=None, cap=0.0,
                     dtype=torch.bfloat16):
    """O, LSE and their tolerances: those of :func:`tree_attention` over caches that begin with the prefix pk, pv [Hkv, P,
    D], its P rows among the cached ones."""
    B, P = q.shape[0], pk.shape[1]
    k, v = (torch.cat((x[None].expand(B, -1, -1, -1), y), dim=2) for x, y in ((pk, kc), (pv, vc)))
    fits = [0 <= int(n) <= kc.shape[2] - q.shape[2] for n in lengths]
    n = torch.tensor([P + int(n) if ok else -1 for n, ok in zip(lengths, fits)])
    return tree_attention(q, k, v, n, mask, window, depths, scale, cap, dtype)
