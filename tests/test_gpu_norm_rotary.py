"""Norm and rotation of each head on the GPU, and the appends behind it, against the float64 oracle, element by element
with the tolerance that follows from the kernel's arithmetic (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc
from test_gpu_rotary import draw, pos_of, within

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def weight(seed, D, dtype):
    return (1.0 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


CASES = [
    # dtype, weights, B, Hq, Hkv, S, D, pairs, interleaved, positions, layout
    (BF, BF, 2, 4, 2, 67, 128, 64, False, "none", "bnsd"),
    (BF, FS, 2, 4, 2, 67, 128, 64, True, "batch", "bsnd"),
    (FH, FH, 1, 7, 1, 1, 64, 32, False, "far", "bnsd"),
    (FH, FS, 3, 5, 5, 33, 64, 16, True, "strided", "padded"),
    (FH, FH, 1, 3, 1, 130, 256, 32, False, "batch", "odd"),
    (FS, FS, 2, 3, 1, 40, 128, 32, True, "far", "bnsd"),
    (FS, FS, 1, 2, 2, 513, 32, 16, False, "far", "bsnd"),
    (FS, FS, 1, 2, 1, 9, 256, 128, False, "batch", "padded"),
    (BF, BF, 1, 2, 1, 300, 32, 8, True, "none", "bnsd"),
    # pairs that do not fill 16 bytes, none at all
    (BF, FS, 2, 3, 1, 50, 64, 5, False, "batch", "bnsd"),
    (FH, FH, 1, 2, 2, 31, 128, 63, True, "none", "bsnd"),
    (FS, FS, 1, 2, 2, 31, 32, 1, False, "far", "bnsd"),
    (FS, FS, 1, 1, 1, 5, 256, 30, True, "strided", "padded"),
    (BF, BF, 1, 2, 1, 20, 32, 3, False, "none", "bnsd"),
    (BF, BF, 1, 2, 1, 20, 128, 0, False, "none", "bnsd"),
    # more heads than a thread takes at once, many tokens
    (BF, BF, 1, 37, 3, 1100, 64, 32, False, "none", "bnsd"),
]


def made(i):
    dtype, wt, B, Hq, Hkv, S, D, pairs, inter, pos, layout = CASES[i]
    q, k = draw(i, B, Hq, S, D, dtype, layout) * 3, draw(100 + i, B, Hkv, S, D, dtype, layout)
    f = rot.rotary_frequencies(2 * pairs, scaling="yarn", factor=4.0, original_length=512, device="cuda") if pairs else \
        (torch.empty(0, dtype=torch.float64, device="cuda"), 1.0)
    return q, k, weight(400 + i, D, wt), weight(500 + i, D, wt), *f, *pos_of(pos, B, S)


@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward_and_gradients(gpu_device, i):
    dtype, wt, B, Hq, Hkv, S, D, pairs, inter, _, layout = CASES[i]
    q, k, wq, wk, f, m, dev, host = made(i)
    gq, gk = draw(200 + i, B, Hq, S, D, dtype, layout), draw(300 + i, B, Hkv, S, D, dtype)
    for x in (q, k, wq, wk):
        x.requires_grad_()
    eps = 1e-5
    y = rot.norm_rotary_embedding(q, k, wq, wk, f, positions=dev, interleaved=inter, magnitude=m, eps=eps)
    d = torch.autograd.grad(y, (q, wq, k, wk), (gq, gk))
    for j, (what, x, w, g) in enumerate((("q", q, wq, gq), ("k", k, wk, gk))):
        x64, w64 = x.detach().cpu().double(), w.detach().cpu().double()
        assert y[j].dtype == dtype and y[j].shape == x.shape and d[2 * j].dtype == dtype and d[2 * j + 1].dtype == wt
        ref, slack = orc.norm_rotary(x64, w64, f.cpu(), host, inter, m, eps)
        within(y[j], ref, orc.rounded(ref, slack, dtype), what)
        (dx, sx), (dw, sw) = orc.norm_rotary_grad(x64, w64, g.cpu().double(), f.cpu(), host, inter, m, eps)
        within(d[2 * j], dx, orc.rounded(dx, sx, dtype), "d" + what)
        within(d[2 * j + 1], dw, orc.rounded(dw, sw, wt), "dw" + what)


@pytest.mark.parametrize("i", [0, 9, 15])
def test_deterministic(gpu_device, i):
    dtype, wt, B, Hq, Hkv, S, D, pairs, inter, _, layout = CASES[i]
    q, k, wq, wk, f, m, dev, _ = made(i)
    gq, gk = draw(200 + i, B, Hq, S, D, dtype), draw(300 + i, B, Hkv, S, D, dtype)
    for x in (q, k, wq, wk):
        x.requires_grad_()
    outs = []
    for _ in range(2):
        y = rot.norm_rotary_embedding(q, k, wq, wk, f, positions=dev, interleaved=inter, magnitude=m)
        outs.append(y + torch.autograd.grad(y, (q, k, wq, wk), (gq, gk)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_against_differences(gpu_device, inter):
    """fp32: (f(x + h d) - f(x - h d)) / 2h along a random direction of all four inputs is the gradient's component along
    it, up to the difference's own truncation, which the oracle's difference in 64 bits has too, and f's rounding over h:
    2^-19 of the sum of |y g| each."""
    xs = [draw(1, 1, 2, 13, 64, FS), draw(2, 1, 1, 13, 64, FS), weight(3, 64, FS), weight(4, 64, FS)]
    gs = draw(5, 1, 2, 13, 64, FS), draw(6, 1, 1, 13, 64, FS)
    ds = [0.1 * draw(7, 1, 2, 13, 64, FS), 0.1 * draw(8, 1, 1, 13, 64, FS), 0.1 * weight(9, 64, FS), 0.1 * weight(10, 64, FS)]
    f, _ = rot.rotary_frequencies(48, device="cuda")
    h = 2.0 ** -5

    def kernel(a, b, u, v):
        return rot.norm_rotary_embedding(a, b, u, v, f, interleaved=inter)

    def oracle(a, b, u, v):
        at = torch.arange(13)[None]
        return tuple(orc.norm_rotary(x.cpu().double(), w.cpu().double(), f.cpu(), at, inter)[0].cuda()
                     for x, w in ((a, u), (b, v)))

    def loss(run, t):
        return sum((y.double() * g).sum() for y, g in zip(run(*[x.double() + t * d for x, d in zip(xs, ds)] if run is oracle
                                                              else [x + t * d for x, d in zip(xs, ds)]), gs))

    leaves = [x.clone().requires_grad_() for x in xs]
    grads = torch.autograd.grad(kernel(*leaves), leaves, gs)
    along = sum((g.double() * d).sum() for g, d in zip(grads, ds)).item()
    diff = ((loss(kernel, h) - loss(kernel, -h)) / (2 * h)).item()
    exact = ((loss(oracle, 2.0 ** -12) - loss(oracle, -2.0 ** -12)) * 2.0 ** 11).item()
    cut = abs(((loss(oracle, h) - loss(oracle, -h)) / (2 * h)).item() - exact)
    size = sum((y.abs() * g.abs()).double().sum() for y, g in zip(kernel(*xs), gs)).item()
    # (inputs x + t d are rounded once, 2^-24 of them, as much again as one of f's own steps)
    assert abs(along - diff) <= 1.01 * cut + size * 2.0 ** -18 / h
    assert abs(along) > 10 * (1.01 * cut + size * 2.0 ** -18 / h)  # (what is compared is larger than what it may be off)


def test_one_output_broadcast_and_frozen_weights(gpu_device):
    q, k = draw(1, 2, 2, 9, 32, FS).requires_grad_(), draw(2, 1, 1, 9, 32, FS).requires_grad_()
    wq, wk = weight(3, 32, FS), weight(4, 32, FS).requires_grad_()
    f, _ = rot.rotary_frequencies(32, device="cuda")
    y, z = rot.norm_rotary_embedding(q, k.expand(2, 3, 9, 32), wq, wk, f)  # one key head for three, and both sequences
    g = draw(3, 2, 3, 9, 32, FS)
    dk, dw = torch.autograd.grad(z, (k, wk), g, retain_graph=True)
    (dx, sx), (dv, sv) = orc.norm_rotary_grad(k.detach().cpu().double().expand(2, 3, 9, 32), wk.detach().cpu().double(),
                                              g.cpu().double(), f.cpu(), torch.arange(9).expand(2, 9))
    # six fp32 terms are added: 5 roundings of at most the sum of magnitudes
    tol = orc.rounded(dx, sx, FS).sum(dim=(0, 1), keepdim=True) + dx.abs().sum(dim=(0, 1), keepdim=True) * 5 * 2.0 ** -24
    within(dk, dx.sum(dim=(0, 1), keepdim=True), tol, "dk of a broadcast key")
    within(dw, dv, orc.rounded(dv, sv, FS), "dw")
    gq = draw(4, 2, 2, 9, 32, FS)
    dq, = torch.autograd.grad(y, q, gq, retain_graph=True)
    (dx, sx), _ = orc.norm_rotary_grad(q.detach().cpu().double(), wq.cpu().double(), gq.cpu().double(), f.cpu(),
                                       torch.arange(9).expand(2, 9))
    within(dq, dx, orc.rounded(dx, sx, FS), "dq")
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y, q, gq, create_graph=True)
    y2, none = rot.norm_rotary_embedding(q, None, wq, None, f)
    assert none is None and torch.equal(y2, y)


def test_rows_without_size_and_not_numbers(gpu_device):
    """A row of zeros stays zeros, with finite gradients; a NaN stays in its row; half an underflowing square counts as 0."""
    q = draw(1, 1, 2, 6, 64, BF)
    q[0, 0, 2] = 0.0
    q[0, 1, 3, 7] = float("nan")
    q.requires_grad_()
    w = weight(2, 64, FS).requires_grad_()
    f, _ = rot.rotary_frequencies(64, device="cuda")
    y, _ = rot.norm_rotary_embedding(q, None, w, None, f)
    dq, = torch.autograd.grad(y, q, torch.ones_like(y))
    assert bool((y[0, 0, 2] == 0).all()) and bool(torch.isfinite(dq[0, 0]).all())
    assert bool(torch.isnan(y[0, 1, 3]).all())
    y = y.detach().clone()
    y[0, 1, 3] = 0
    assert bool(torch.isfinite(y).all())


def test_empty_inputs_and_refusals(gpu_device):
    f, _ = rot.rotary_frequencies(64, device="cuda")
    w = weight(1, 64, BF)
    e = draw(1, 1, 2, 0, 64, BF).requires_grad_()
    wr = w.clone().requires_grad_()
    y, z = rot.norm_rotary_embedding(e, e, wr, w, f)
    assert y.shape == z.shape == (1, 2, 0, 64)
    dw, = torch.autograd.grad(y, wr, torch.zeros_like(y))
    assert bool((dw == 0).all())
    q = draw(1, 1, 2, 4, 64, BF)
    ok = dict(query_weight=w, key_weight=w, inv_freq=f)
    for kw in (dict(inv_freq=f.cpu()), dict(inv_freq=f.float()), dict(positions=torch.arange(4)), dict(magnitude=float("inf")),
               dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(query_weight=w.half()),
               dict(query_weight=w[:32]), dict(query_weight=w.float()), dict(key_weight=None), dict(key_weight=w.cpu()),
               dict(query_weight=w[None])):
        with pytest.raises(RuntimeError):
            rot.norm_rotary_embedding(q, q, **dict(ok, **kw))
    with pytest.raises(RuntimeError):
        rot.norm_rotary_embedding(q, q.half(), **ok)
    with pytest.raises(RuntimeError):
        rot.norm_rotary_embedding(q, None, **ok)
    with pytest.raises(AssertionError):
        rot.norm_rotary_embedding(q, q[:, :, :2], **ok)
    with pytest.raises(AssertionError):
        rot.norm_rotary_embedding(q[:, :0], q, **ok)


def test_on_another_stream_and_in_a_graph(gpu_device):
    """Captured forward and backward replay to the eager results as inputs and weights change."""
    f, m = rot.rotary_frequencies(64, device="cuda")
    q, k = draw(1, 2, 4, 33, 64, BF), draw(2, 2, 2, 33, 64, BF)
    wq, wk = weight(3, 64, BF), weight(4, 64, BF)
    gq, gk = draw(5, 2, 4, 33, 64, BF), draw(6, 2, 2, 33, 64, BF)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]

    def step():
        y = rot.norm_rotary_embedding(q, k, wq, wk, f, magnitude=m)
        return list(y) + list(torch.autograd.grad(y, leaves, (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            first = [x.detach().clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        with torch.no_grad():
            q.copy_(draw(10 + turn, 2, 4, 33, 64, BF))
            wk.copy_(weight(20 + turn, 64, BF))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in out]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        want = None
    assert len(first) == 6


APPENDS = [
    # dtype, weights, B, Hq, Hkv, S, C, D, pairs, interleaved, layout, lengths
    (BF, BF, 3, 4, 2, 1, 50, 128, 64, False, "bnsd", [0, 49, 20]),
    (FH, FS, 2, 3, 1, 5, 64, 64, 10, True, "bsnd", [59, 3]),
    (FS, FS, 2, 2, 2, 7, 40, 32, 16, False, "odd", [36, 40]),        # rows outside the cache are not written
    (BF, FS, 1, 5, 1, 300, 320, 256, 0, False, "padded", [11]),
]


@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(gpu_device, i):
    dtype, wt, B, Hq, Hkv, S, C, D, pairs, inter, layout, n = APPENDS[i]
    q, k, v = (draw(s + i, B, h, S, D, dtype, layout) for s, h in ((0, Hq), (40, Hkv), (80, Hkv)))
    kc, vc = draw(120 + i, B, Hkv, C, D, dtype), draw(160 + i, B, Hkv, C, D, dtype)
    wq, wk = weight(1, D, wt), weight(2, D, wt)
    old = kc.clone(), vc.clone()
    f = rot.rotary_frequencies(2 * pairs, device="cuda")[0] if pairs else None
    f64 = f.cpu() if pairs else torch.empty(0, dtype=torch.float64)
    y = fc.norm_rotary_append(q, k, v, kc, vc, torch.tensor(n, dtype=torch.int32, device="cuda"), wq, wk, f,
                              interleaved=inter, eps=1e-4)
    host = torch.tensor(n)[:, None] + torch.arange(S)
    ref, slack = orc.norm_rotary(q.cpu().double(), wq.cpu().double(), f64, host, inter, 1.0, 1e-4)
    within(y, ref, orc.rounded(ref, slack, dtype), "q")
    ref, slack = orc.norm_rotary(k.cpu().double(), wk.cpu().double(), f64, host, inter, 1.0, 1e-4)
    tol = orc.rounded(ref, slack, dtype)
    for b in range(B):
        rows = [s for s in range(S) if n[b] + s < C]
        at = [n[b] + s for s in rows]
        within(kc[b, :, at], ref[b, :, rows], tol[b, :, rows], "k")
        assert torch.equal(vc[b, :, at], v[b, :, rows])
        rest = [r for r in range(C) if r not in at]
        assert torch.equal(kc[b, :, rest], old[0][b, :, rest]) and torch.equal(vc[b, :, rest], old[1][b, :, rest])
    kc2, vc2 = old[0].clone(), old[1].clone()
    none = fc.norm_rotary_append(q[:, :0], k, v, kc2, vc2, torch.tensor(n, dtype=torch.int32, device="cuda"), wq, wk, f,
                                 interleaved=inter, eps=1e-4)  # keys and values alone
    assert none.shape == (B, 0, S, D) and torch.equal(kc2, kc) and torch.equal(vc2, vc)
