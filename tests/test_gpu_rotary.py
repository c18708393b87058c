"""Rotary positions and cache appends on the GPU against the float64 oracle, element by element with the tolerance that
follows from the kernel's arithmetic (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def within(x, y, tol, what=""):
    x = x.detach().cpu().double()
    bad = (x - y).abs() > tol
    assert not bool(bad.any()) and bool(torch.isfinite(x).all()), \
        f"{what}: {int(bad.sum())} of {bad.numel()}, worst {((x - y).abs() / tol).max().item():.2f} tolerances"


def draw(seed, B, H, S, D, dtype, layout="bnsd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "bsnd":
        return torch.randn(B, S, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    if layout == "padded":  # rows on 16-byte boundaries, longer than the head
        return torch.randn(B, H, S, D + 16, generator=g).to(dtype).cuda()[..., 8:8 + D]
    if layout == "odd":     # rows off 16-byte boundaries: copied by the call
        return torch.randn(B, H, S, D + 1, generator=g).to(dtype).cuda()[..., 1:]
    return torch.randn(B, H, S, D, generator=g).to(dtype).cuda()


def pos_of(kind, B, S):
    if kind == "none":
        return None, torch.arange(S).expand(B, S)
    if kind == "far":   # one row of positions, far out
        p = torch.arange(S) + 1048576 - S
        return p.cuda(), p.expand(B, S)
    if kind == "batch":  # each sequence its own, in no order, some negative
        p = torch.randint(-5000, 200000, (B, S), generator=torch.Generator().manual_seed(9), dtype=torch.int32)
        return p.cuda(), p
    p = torch.randint(0, 9000, (S, 2 * B), generator=torch.Generator().manual_seed(9)).cuda()[:, ::2].t()  # "strided"
    return p, p.cpu()


CASES = [
    # dtype, B, Hq, Hkv, S, D, pairs, interleaved, positions, layout
    (BF, 2, 4, 2, 67, 128, 64, False, "none", "bnsd"),
    (BF, 2, 4, 2, 67, 128, 64, True, "batch", "bsnd"),
    (FH, 1, 7, 1, 1, 64, 32, False, "far", "bnsd"),
    (FH, 3, 5, 5, 33, 64, 16, True, "strided", "padded"),
    (FH, 1, 3, 1, 130, 256, 32, False, "batch", "odd"),
    (FS, 2, 3, 1, 40, 128, 32, True, "far", "bnsd"),
    (FS, 1, 2, 2, 513, 32, 16, False, "far", "bsnd"),
    (FS, 1, 2, 1, 9, 256, 128, False, "batch", "padded"),
    (BF, 1, 2, 1, 300, 32, 8, True, "none", "bnsd"),
    # pairs that do not fill 16 bytes: the general kernel
    (BF, 2, 3, 1, 50, 64, 5, False, "batch", "bnsd"),
    (FH, 1, 2, 2, 31, 128, 63, True, "none", "bsnd"),
    (FS, 1, 2, 2, 31, 32, 1, False, "far", "bnsd"),
    (FS, 1, 1, 1, 5, 64, 30, True, "strided", "padded"),
    # more heads than a thread takes at once, many tokens
    (BF, 1, 37, 3, 1100, 64, 32, False, "none", "bnsd"),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward_and_gradients(gpu_device, i):
    dtype, B, Hq, Hkv, S, D, pairs, inter, pos, layout = CASES[i]
    q, k = draw(i, B, Hq, S, D, dtype, layout), draw(100 + i, B, Hkv, S, D, dtype, layout)
    gq, gk = draw(200 + i, B, Hq, S, D, dtype, layout), draw(300 + i, B, Hkv, S, D, dtype)
    f, m = rot.rotary_frequencies(2 * pairs, scaling="yarn", factor=4.0, original_length=512, device="cuda")
    dev, host = pos_of(pos, B, S)
    q.requires_grad_()
    k.requires_grad_()
    yq, yk = rot.rotary_embedding(q, k, f, positions=dev, interleaved=inter, magnitude=m)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for what, x, y, inv in (("q", q, yq, False), ("k", k, yk, False), ("dq", gq, dq, True), ("dk", gk, dk, True)):
        assert y.dtype == dtype and y.shape == x.shape
        ref, slack = orc.rotary(x.detach().cpu().double(), f.cpu(), host, inter, m, inv)
        within(y, ref, orc.rounded(ref, slack, dtype), what)
        assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])  # the rest is a copy


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_against_differences(gpu_device, inter):
    """fp32: (f(x + h d) - f(x - h d)) / 2h along a random direction is the gradient's component along it.  f is linear,
    so the difference has no truncation error: its rounding, about 2^-22 of the sum of |y g| over h = 1/4, remains."""
    q, k = draw(1, 1, 2, 13, 64, FS).requires_grad_(), draw(2, 1, 1, 13, 64, FS).requires_grad_()
    gq, gk = draw(3, 1, 2, 13, 64, FS), draw(4, 1, 1, 13, 64, FS)
    d1, d2 = draw(5, 1, 2, 13, 64, FS), draw(6, 1, 1, 13, 64, FS)
    f, _ = rot.rotary_frequencies(48, device="cuda")

    def loss(a, b):
        y, z = rot.rotary_embedding(a, b, f, interleaved=inter)
        return (y.double() * gq).sum() + (z.double() * gk).sum()

    dq, dk = torch.autograd.grad(loss(q, k), (q, k))
    along = ((dq * d1).double().sum() + (dk * d2).double().sum()).item()
    h = 0.25
    with torch.no_grad():
        diff = ((loss(q + h * d1, k + h * d2) - loss(q - h * d1, k - h * d2)) / (2 * h)).item()
        size = 2 * ((q.abs() + d1.abs()).double().sum() * gq.abs().max() + (k.abs() + d2.abs()).double().sum()
                    * gk.abs().max()).item()
    assert abs(along - diff) <= size * 2.0 ** -22 / h


def test_gradients_of_one_output_broadcast_inputs_and_twice(gpu_device):
    q, k = draw(1, 2, 2, 9, 32, FS).requires_grad_(), draw(2, 1, 1, 9, 32, FS).requires_grad_()
    f, _ = rot.rotary_frequencies(32, device="cuda")
    y, z = rot.rotary_embedding(q, k.expand(2, 3, 9, 32), f)  # one key head for three, and for both sequences
    g = draw(3, 2, 3, 9, 32, FS)
    dk, = torch.autograd.grad(z, k, g, retain_graph=True)
    ref, slack = orc.rotary(g.cpu().double(), f.cpu(), torch.arange(9).expand(2, 9), inverse=True)
    # six fp32 terms are added: 5 roundings of at most the sum of magnitudes
    tol = orc.rounded(ref, slack, FS).sum(dim=(0, 1), keepdim=True) + ref.abs().sum(dim=(0, 1), keepdim=True) * 5 * 2.0 ** -24
    within(dk, ref.sum(dim=(0, 1), keepdim=True), tol, "dk of a broadcast key")
    dq, none = torch.autograd.grad(y, (q, k), draw(4, 2, 2, 9, 32, FS), allow_unused=True, create_graph=True)
    assert none is None or float(none.abs().max()) == 0.0
    q2 = draw(5, 2, 2, 9, 32, FS).requires_grad_()
    y2, no_key = rot.rotary_embedding(q2, None, f)
    assert no_key is None
    w = draw(6, 2, 2, 9, 32, FS).requires_grad_()
    d1, = torch.autograd.grad(y2, q2, w, create_graph=True)
    dw, = torch.autograd.grad(d1, w, draw(7, 2, 2, 9, 32, FS))  # the gradient of the gradient turns forward again
    ref, slack = orc.rotary(draw(7, 2, 2, 9, 32, FS).cpu().double(), f.cpu(), torch.arange(9).expand(2, 9))
    within(dw, ref, orc.rounded(ref, slack, FS), "second")


def test_empty_inputs_and_refusals(gpu_device):
    f, _ = rot.rotary_frequencies(64, device="cuda")
    y, z = rot.rotary_embedding(draw(1, 1, 2, 0, 64, BF), draw(1, 1, 2, 0, 64, BF), f)
    assert y.shape == z.shape == (1, 2, 0, 64)
    q = draw(1, 1, 2, 4, 64, BF)
    for kw in (dict(inv_freq=f.cpu()), dict(inv_freq=f.float()), dict(inv_freq=torch.cat((f, f))),
               dict(inv_freq=f, positions=torch.arange(4)), dict(inv_freq=f, positions=torch.arange(3, device="cuda")),
               dict(inv_freq=f, magnitude=float("nan"))):
        with pytest.raises(RuntimeError):
            rot.rotary_embedding(q, q, **kw)
    with pytest.raises(RuntimeError):
        rot.rotary_embedding(q, q.half(), f)
    with pytest.raises(RuntimeError):
        rot.rotary_embedding(draw(1, 1, 2, 4, 96, BF), None, f)
    with pytest.raises(AssertionError):
        rot.rotary_embedding(q, q[:, :, :2], f)


def test_on_another_stream_and_in_a_graph(gpu_device):
    """Captured forward and backward replay to the eager results as inputs and positions change."""
    f, m = rot.rotary_frequencies(64, device="cuda")
    q, k = draw(1, 2, 4, 20, 64, BF).requires_grad_(), draw(2, 2, 2, 20, 64, BF).requires_grad_()
    g, pos = draw(3, 2, 4, 20, 64, BF), torch.arange(20, device="cuda")

    def step(q, k, g, pos):
        y, z = rot.rotary_embedding(q, k, f, positions=pos)
        return (y, z) + torch.autograd.grad((y, z), (q, k), (g, g[:, :2]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.detach().clone() for t in step(q, k, g, pos)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(q, k, g, pos)
    for rep in range(3):
        with torch.no_grad():
            q.copy_(draw(10 + rep, 2, 4, 20, 64, BF))
            pos.add_(77)
        eager = [t.detach().clone() for t in step(q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_(),
                                                  g, pos.clone())]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)
    assert not torch.equal(first[0], outs[0])


APPENDS = [
    # dtype, B, Hq, Hkv, S, C, D, pairs, interleaved, positions, layout, lengths
    (BF, 3, 4, 2, 1, 50, 128, 64, False, False, "bnsd", [0, 49, 20]),
    (FH, 2, 7, 1, 30, 64, 64, 16, True, True, "bsnd", [34, 0]),
    (FS, 2, 2, 2, 9, 40, 32, 3, False, False, "odd", [5, 31]),
    (BF, 2, 2, 1, 130, 300, 256, 0, False, False, "padded", [10, 170]),
    # rows behind the end, and before the beginning, of the cache are not written
    (BF, 4, 2, 2, 5, 16, 64, 32, False, False, "bnsd", [14, 16, -3, 2000000000]),
]


@pytest.mark.parametrize("inter_cache", [False, True])
@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(gpu_device, i, inter_cache):
    dtype, B, Hq, Hkv, S, C, D, pairs, inter, given, layout, n = APPENDS[i]
    q, k, v = (draw(j, B, h, S, D, dtype, layout) for j, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    if inter_cache:  # [B, C, K or V, H, D]: keys and values of a token side by side
        both = draw(4, B * C, 2 * Hkv, 1, D, dtype).reshape(B, C, 2, Hkv, D)
        kc, vc = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    else:
        kc, vc = draw(4, B, Hkv, C, D, dtype), draw(5, B, Hkv, C, D, dtype)
    k0, v0 = kc.cpu(), vc.cpu()
    f, m = rot.rotary_frequencies(2 * pairs, device="cuda") if pairs else (None, 1.0)
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    rows = torch.tensor(n)[:, None] + torch.arange(S)
    pos = torch.randint(0, 4000, (B, S), generator=torch.Generator().manual_seed(1)) if given else rows
    out = fc.rotary_append(q, k, v, kc, vc, lengths, f, positions=pos.cuda() if given else None, interleaved=inter)
    fr = torch.zeros(0, dtype=torch.float64) if f is None else f.cpu()
    ref, slack = orc.rotary(q.cpu().double(), fr, pos, inter)
    within(out, ref, orc.rounded(ref, slack, dtype), "q")
    kr, ks = orc.rotary(k.cpu().double(), fr, pos, inter)
    kt = orc.rounded(kr, ks, dtype)
    want_k, want_v, tol = k0.double(), v0.clone(), torch.zeros(B, Hkv, C, D, dtype=torch.float64)
    for b in range(B):
        for s in range(S):
            j = n[b] + s
            if 0 <= j < C:
                want_k[b, :, j], tol[b, :, j], want_v[b, :, j] = kr[b, :, s], kt[b, :, s], v.cpu()[b, :, s]
    within(kc, want_k, tol, "key cache")
    assert torch.equal(vc.cpu(), want_v)
    assert lengths.tolist() == n


def test_append_refusals(gpu_device):
    q, c = draw(1, 1, 2, 3, 64, BF), draw(2, 1, 2, 20, 64, BF)
    n = torch.tensor([4], dtype=torch.int32, device="cuda")
    f, _ = rot.rotary_frequencies(64, device="cuda")
    with pytest.raises(RuntimeError, match="written in place"):
        fc.rotary_append(q, q, q, draw(2, 1, 2, 20, 64, BF, "odd"), c, n, f)
    with pytest.raises(RuntimeError):
        fc.rotary_append(q, q, q, c, c[:, :1].expand(1, 2, 20, 64), n, f)  # heads that share their rows
    with pytest.raises(RuntimeError):
        fc.rotary_append(q, c[:, :, :3], q, c, c.clone(), n, f)            # tokens inside the cache
    with pytest.raises(RuntimeError, match="gradient"):
        fc.rotary_append(q.clone().requires_grad_(), q, q, c, c.clone(), n, f)
    with pytest.raises(RuntimeError, match="lengths"):
        fc.rotary_append(q, q, q, c, c.clone(), n.cpu(), f)
    with pytest.raises(AssertionError):
        fc.rotary_append(q, q[:, :1], q, c, c.clone(), n, f)
    y = fc.rotary_append(q[:, :, :0], q[:, :, :0], q[:, :, :0], c, c.clone(), n, f)
    assert y.shape == (1, 2, 0, 64)
