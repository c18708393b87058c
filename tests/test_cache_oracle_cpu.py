"""The bounds of the cache oracle (oracle/cache_oracle.py) on the host: far below the outputs that they are for, so that an
output which lost a part of its keys, or all of them, is outside; and what the kernels' roundings do stays inside."""
import pytest
import torch

from oracle import cache_oracle as orc

BF, FH = torch.bfloat16, torch.float16
F8, I8 = torch.float8_e4m3fn, torch.int8


def rms(x):
    return x.square().mean().sqrt().item()


def cache(seed, B, H, C, D, kind, spread):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, C, D, generator=g) * torch.exp(spread * torch.randn(B, H, C, 1, generator=g))
    s = (x.abs().amax(dim=-1) / orc.TOP[kind]).float()
    y = x / s[..., None]
    return (y.round().to(I8) if kind == I8 else y.to(F8)), s


LONG = [
    # dtype, cache, Hq, Hkv, T, C, D, length
    (BF, F8, 4, 1, 2, 9000, 128, 8998), (FH, I8, 2, 1, 1, 20000, 128, 19999), (FH, F8, 2, 1, 20, 9000, 64, 8000),
    (BF, I8, 2, 1, 4, 20000, 64, 19000), (FH, F8, 1, 1, 3, 2000, 256, 1990), (BF, I8, 2, 1, 1, 300, 32, 299),
]


def made(i):
    dtype, kind, Hq, Hkv, T, C, D, n = LONG[i]
    q = torch.randn(1, Hq, T, D, generator=torch.Generator().manual_seed(i)).to(dtype)
    return (q, *(x for s, p in ((50, 0.3), (90, 1.0)) for x in cache(s + i, 1, Hkv, C, D, kind, p))), n, dtype


@pytest.mark.parametrize("i", range(len(LONG)))
def test_bounds_over_8_bits_are_far_below_the_output(i):
    (q, kc, ks, vc, vs), n, dtype = made(i)
    o, lse, to, tl = orc.quantized_tree_attention(q, kc, vc, ks, vs, [n], dtype=dtype)
    assert rms(to) <= rms(o) / 8 and bool((tl < 2e-3).all())
    lost = vc.clone()
    lost[:, :, : n // 8] = 0  # an eighth of the keys without values
    part = orc.quantized_tree_attention(q, kc, lost, ks, vs, [n], dtype=dtype)[0]
    assert ((part - o).abs() > to).double().mean() > 0.25


@pytest.mark.parametrize("i,rest", [(i, rest) for i in range(len(LONG)) for rest in (False, True)
                                    if not rest or LONG[i][0] == FH])
def test_rounded_weights_are_within_the_bounds(i, rest):
    """Weights times scales in fp16 as the kernel holds them, with what that leaves and without: what is within the bounds
    (fp16 queries without the rest are not), and the error against that of rounding the output alone."""
    (q, kc, ks, vc, vs), n, dtype = made(i)
    o, _, to, _ = orc.quantized_tree_attention(q, kc, vc, ks, vs, [n], dtype=dtype)
    G, N = q.shape[1] // kc.shape[1], n + q.shape[2]
    got = torch.zeros_like(o)
    for h in range(q.shape[1]):
        k, c, s = kc[0, h // G, :N].double() * ks[0, h // G, :N].double()[:, None], vc[0, h // G, :N].double(), vs[0, h // G, :N]
        x = q[0, h].double() @ k.T / q.shape[3] ** 0.5
        ok = torch.arange(N)[None] <= n + torch.arange(q.shape[2])[:, None]
        p = torch.exp(x.masked_fill(~ok, float("-inf")) - x.amax(dim=-1, keepdim=True))
        unit = 2.0 ** (6 - torch.floor(torch.log2(s.max().double())))
        w = p * s.double() * unit
        first = w.half().double()
        second = (w - first).half().double() if rest else 0.0
        got[0, h] = (first + second) @ c / unit / p.sum(dim=-1, keepdim=True)
    assert bool(((got - o).abs() <= to).all()) or (dtype == FH and not rest)
    ratio = rms(got.to(dtype).double() - o) / rms(o.to(dtype).double() - o)
    assert ratio <= 1.05 if dtype == BF or rest else ratio > 1.15


TREES = [
    # dtype, Hq, Hkv, T, P, C, D, length
    (BF, 4, 1, 2, 8000, 1100, 128, 1000), (FH, 2, 1, 1, 16383, 700, 128, 600), (FH, 2, 1, 20, 5000, 300, 64, 256),
    (BF, 2, 1, 4, 100, 20000, 64, 19000), (torch.float32, 1, 1, 3, 2000, 300, 256, 290), (FH, 2, 1, 1, 1, 300, 32, 299),
]


@pytest.mark.parametrize("i", range(len(TREES)))
def test_bounds_of_tree_and_prefix_are_far_below_the_output(i):
    """bf16's weights are off by half a step of 2^-8, which is what its bound is for many keys: half of the output."""
    dtype, Hq, Hkv, T, P, C, D, n = TREES[i]
    g = torch.Generator().manual_seed(i)
    q, pk, pv, kc, vc = (torch.randn(*s, D, generator=g).to(dtype)
                         for s in ((1, Hq, T), (Hkv, P), (Hkv, P), (1, Hkv, C), (1, Hkv, C)))
    o, lse, to, tl = orc.prefix_attention(q, pk, pv, kc, vc, [n], dtype=dtype)
    assert rms(to) <= rms(o) / (2 if dtype == BF else 8) and bool((tl < 2e-3).all())
    k, v = torch.cat((pk[None], kc), dim=2), torch.cat((pv[None], vc), dim=2)
    same = orc.tree_attention(q, k, v, [P + n], dtype=dtype)
    assert all(torch.equal(a, b) for a, b in zip((o, lse, to, tl), same))
    x = (q[0].double().unflatten(0, (Hkv, Hq // Hkv)) @ k[0, :, None, :P + n + T].double().transpose(-1, -2)) / D ** 0.5
    ok = torch.arange(P + n + T)[None] <= P + n + torch.arange(T)[:, None]
    p = torch.exp(x.masked_fill(~ok, float("-inf")) - x.amax(dim=-1, keepdim=True))
    w = p.double() if dtype == torch.float32 else p.to(dtype).double()
    got = (w @ v[0, :, None, :P + n + T].double() / p.sum(dim=-1, keepdim=True)).flatten(0, 1)[None]
    assert bool(((got - o).abs() <= to).all())
