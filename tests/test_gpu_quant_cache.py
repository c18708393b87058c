"""A cache of 8 bits written and read back on the GPU against the float64 oracle (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc
from test_gpu_norm_rotary import weight
from test_gpu_rotary import draw, within

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
F8, I8 = torch.float8_e4m3fn, torch.int8


def codes(seed, shape, kind):
    """Any codes but NaN."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 256, shape, generator=g, dtype=torch.int32)
    if kind == F8:
        c[(c & 127) == 127] = 3
    return c.to(torch.uint8).cuda().view(kind)


def caches(seed, B, H, C, D, kind):
    s = torch.rand(2, B, H, C, generator=torch.Generator().manual_seed(seed)).cuda() + 0.01
    return codes(seed, (B, H, C, D), kind), codes(seed + 1, (B, H, C, D), kind), s[0].clone(), s[1].clone()


APPENDS = [
    # dtype, cache, weights, B, Hq, Hkv, S, C, D, pairs, interleaved, layout, lengths
    (BF, F8, BF, 3, 4, 2, 1, 50, 128, 64, False, "bnsd", [0, 49, 20]),
    (BF, I8, FS, 3, 4, 2, 1, 50, 128, 64, True, "bnsd", [0, 49, 20]),
    (FH, F8, None, 2, 3, 1, 5, 64, 64, 10, True, "bsnd", [59, 3]),
    (FH, I8, None, 2, 3, 1, 5, 64, 64, 9, False, "bsnd", [59, 3]),
    (FS, F8, FS, 2, 2, 2, 7, 40, 32, 16, False, "odd", [36, 40]),        # rows outside the cache are not written
    (FS, I8, None, 2, 2, 2, 7, 40, 32, 4, True, "odd", [36, -3]),
    (BF, I8, FS, 1, 5, 1, 300, 320, 256, 0, False, "padded", [11]),
    (FS, I8, None, 1, 5, 1, 30, 32, 256, 7, True, "padded", [2]),
    (BF, F8, None, 1, 4, 4, 33, 100, 32, 16, False, "bnsd", [60]),
    (FH, F8, FH, 1, 2, 1, 9, 16, 256, 128, True, "bnsd", [7]),
]


def bits(x):
    return x.view(torch.uint8)


@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(gpu_device, i):
    dtype, kind, wt, B, Hq, Hkv, S, C, D, pairs, inter, layout, n = APPENDS[i]
    q, k, v = (draw(s + i, B, h, S, D, dtype, layout) for s, h in ((0, Hq), (40, Hkv), (80, Hkv)))
    kc, vc, ks, vs = caches(i, B, Hkv, C, D, kind)
    w = dict(query_weight=weight(1, D, wt), key_weight=weight(2, D, wt), eps=1e-4) if wt else {}
    old = [x.clone() for x in (bits(kc), bits(vc), ks, vs)]
    f = rot.rotary_frequencies(2 * pairs, device="cuda")[0] if pairs else None
    f64 = f.cpu() if pairs else torch.empty(0, dtype=torch.float64)
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    y = fc.quantized_append(q, k, v, kc, vc, ks, vs, lengths, f, interleaved=inter, **w)
    host = torch.tensor(n)[:, None] + torch.arange(S)

    def turned(x, name):
        x = x.cpu().double()
        if wt:
            return orc.norm_rotary(x, w[name].cpu().double(), f64, host, inter, 1.0, 1e-4)
        return orc.rotary(x, f64, host, inter)

    ref, slack = turned(q, "query_weight")
    within(y, ref, orc.rounded(ref, slack, dtype), "q")
    ref, slack = turned(k, "key_weight")
    v64 = v.cpu().double()
    for what, cache, scales, want, off, j in (("k", kc, ks, ref, slack, 0), ("v", vc, vs, v64, torch.zeros_like(v64), 1)):
        size = orc.scale_of(want, kind)
        for b in range(B):
            rows = [s for s in range(S) if 0 <= n[b] + s < C]
            at = [n[b] + s for s in rows]
            got, s = scales[b, :, at].cpu().double(), size[b, :, rows]
            assert bool(((got - s).abs() <= s * 2.0 ** -23 + off[b, :, rows].amax(dim=-1) / orc.TOP[kind]).all())
            tol = orc.code_tolerance(want[b, :, rows], off[b, :, rows], got, kind)
            within(cache[b, :, at].float().double() * scales[b, :, at].double()[..., None], want[b, :, rows], tol, what)
            rest = [r for r in range(C) if r not in at]
            assert torch.equal(bits(cache)[b, :, rest], old[j][b, :, rest])
            assert torch.equal(scales[b, :, rest], old[2 + j][b, :, rest])
    kc2, vc2, ks2, vs2 = caches(i, B, Hkv, C, D, kind)
    fc.quantized_append(q[:, :0], k, v, kc2, vc2, ks2, vs2, lengths, f, interleaved=inter, **w)  # keys and values alone
    assert all(torch.equal(a, b) for a, b in zip((bits(kc), bits(vc), ks, vs), (bits(kc2), bits(vc2), ks2, vs2)))


@pytest.mark.parametrize("kind", [F8, I8])
def test_codes_are_the_nearest(gpu_device, kind):
    """fp32 values on, and next to, the borders between codes, of a row whose scale is a power of two: exact."""
    top = orc.TOP[kind]
    if kind == I8:
        grid = torch.arange(-127, 128).double()
    else:
        c = torch.arange(0, 127, dtype=torch.uint8).view(F8).double()
        grid = torch.cat((-c.flip(0), c[1:]))
    mid = (grid[1:] + grid[:-1]) / 2
    x = torch.cat((mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), grid))
    x = torch.cat((x, torch.zeros(-x.numel() % 255, dtype=torch.float64))).view(-1, 255)
    x = torch.cat((x, torch.full((x.shape[0], 1), top, dtype=torch.float64)), dim=1).float() / 64  # scale 1 / 64
    S = x.shape[0]
    v = x[None, None].cuda()
    kc, vc, ks, vs = caches(3, 1, 1, S, 256, kind)
    fc.quantized_append(v[:, :0], v, v, kc, vc, ks, vs, torch.zeros(1, dtype=torch.int32, device="cuda"), None)
    y = x.double() * 64
    want = torch.round(y) if kind == I8 else y.float().to(F8).double()
    for c, s in ((kc, ks), (vc, vs)):
        assert bool((s == 1.0 / 64).all())
        assert torch.equal(c[0, 0].float().cpu().double(), want)


@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("dtype", [BF, FH, FS])
def test_rows_without_size_and_not_numbers(gpu_device, kind, dtype):
    """Zeros have a scale and codes of 0; a row with an infinity or NaN reads back as NaN, and only it; the largest and
    smallest numbers have scales that are numbers."""
    x = draw(1, 1, 2, 8, 64, dtype)
    x[0, 0, 1] = 0
    x[0, 0, 2, 3] = float("inf")
    x[0, 1, 2, 63] = float("nan")
    x[0, 1, 4] = torch.finfo(dtype).max
    x[0, 1, 5] = torch.finfo(dtype).tiny
    kc, vc, ks, vs = caches(3, 1, 2, 8, 64, kind)
    fc.quantized_append(x, x, x, kc, vc, ks, vs, torch.zeros(1, dtype=torch.int32, device="cuda"), None)
    k, v = fc.dequantize_cache(kc, vc, ks, vs, torch.tensor([8], dtype=torch.int32, device="cuda"), dtype=FS)
    assert torch.equal(bits(kc), bits(vc)) and torch.equal(torch.isnan(k), torch.isnan(v))
    bad = torch.zeros(2, 8, dtype=torch.bool)
    bad[0, 2] = bad[1, 2] = True
    assert torch.equal(torch.isnan(k[0]).all(-1).cpu(), bad) and torch.equal(torch.isnan(k[0]).any(-1).cpu(), bad)
    assert bool((bits(kc)[0][bad.cuda()] == 0).all()) and bool((k[0, 0, 1] == 0).all())
    big = k[0, 1, 4].double().cpu()
    assert bool(((big / torch.finfo(dtype).max - 1).abs() < 2.0 ** -20).all())


READS = [
    # cache, dtype, B, H, C, D, lengths
    (F8, BF, 2, 3, 50, 128, [50, 17]), (I8, BF, 2, 3, 51, 64, [0, 51]), (F8, FH, 1, 1, 1, 32, [1]),
    (I8, FH, 3, 2, 200, 256, [7, 200, 300]), (F8, FS, 2, 2, 77, 256, [-4, 70]), (I8, FS, 1, 2, 333, 32, [333]),
    (F8, BF, 4, 8, 5000, 128, [5000, 1, 4097, 128]),  # four rows a thread
    (I8, FS, 4, 8, 2500, 64, [2500, 1, 2049, 128]),
]


@pytest.mark.parametrize("i", range(len(READS)))
def test_read_back(gpu_device, i):
    kind, dtype, B, H, C, D, n = READS[i]
    kc, vc, ks, vs = caches(i, B, H, C, D, kind)
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    out = fc.dequantize_cache(kc, vc, ks, vs, lengths, dtype=dtype)
    into = [torch.full((B, H, C + 1, D), 7.0, dtype=dtype, device="cuda")[:, :, :C] for _ in range(2)]
    again = fc.dequantize_cache(kc, vc, ks, vs, lengths, out=(into[0], into[1]))
    assert again[0] is into[0] and again[1] is into[1]
    for x, y, c, s in zip(out, into, (kc, vc), (ks, vs)):
        want = (c.float() * s[..., None]).to(dtype)  # (one product of 32 bits, one rounding)
        assert x.dtype == dtype
        for b in range(B):
            m = min(max(n[b], 0), C)
            assert torch.equal(x[b, :, :m], want[b, :, :m]) and bool((x[b, :, m:] == 0).all())
            assert torch.equal(y[b, :, :m], want[b, :, :m]) and bool((y[b, :, m:] == 7).all())


def test_strided_caches(gpu_device):
    """Keys and values side by side in one buffer, read and written in place; scales of other strides are read, not
    written."""
    both = codes(1, (2, 40, 2, 2, 64), I8)  # [B, C, H, key or value, D]
    kc, vc = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    ks, vs = torch.rand(2, 2, 40, device="cuda"), torch.rand(2, 2, 40, device="cuda")
    x = draw(2, 2, 2, 3, 64, BF)
    n = torch.tensor([5, 37], dtype=torch.int32, device="cuda")
    want = [kc.contiguous(), vc.contiguous(), ks.clone(), vs.clone()]
    fc.quantized_append(x, x, x, *want, n, None)
    fc.quantized_append(x, x, x, kc, vc, ks, vs, n, None)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and torch.equal(ks, want[2]) and torch.equal(vs, want[3])
    ts = ks.transpose(1, 2).contiguous().transpose(1, 2)
    a = fc.dequantize_cache(kc, vc, ts, vs, n + 3)
    b = fc.dequantize_cache(want[0], want[1], ks, vs, n + 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(RuntimeError, match="contiguous"):
        fc.quantized_append(x, x, x, kc, vc, ts, vs, n, None)


def test_refusals(gpu_device):
    x = draw(1, 1, 2, 3, 64, BF)
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    kc, vc, ks, vs = caches(1, 1, 2, 8, 64, F8)
    ok = dict(query=x, key=x, value=x, key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, lengths=n, inv_freq=None)
    w = weight(1, 64, BF)
    for kw in (dict(key_cache=x), dict(value_cache=vc.view(I8)), dict(key_cache=kc.view(torch.uint8)),
               dict(key_scales=ks[:, :1]), dict(value_scales=vs.double()), dict(key_scales=ks.cpu()), dict(key_scales=vs),
               dict(value_cache=kc), dict(query_weight=w), dict(key_weight=w), dict(query_weight=w, key_weight=w, eps=0.0),
               dict(lengths=n.long()), dict(key=x.half()), dict(key_scales=ks.clone().requires_grad_()),
               dict(key_cache=codes(1, (1, 2, 8, 65), F8)[..., 1:])):
        with pytest.raises(RuntimeError):
            fc.quantized_append(**dict(ok, **kw))
    with pytest.raises(AssertionError):
        fc.quantized_append(**dict(ok, value_cache=vc[:, :, :4]))
    for args, kw in (((kc, vc, ks, vs, n), dict(dtype=torch.float64)), ((kc, vc, ks, vs, n), dict(dtype=F8)),
                     ((x, x, ks, vs, n), {}), ((kc, vc, ks, vs[:, :1], n), {}), ((kc, vc, ks, vs, n.cpu()), {}),
                     ((kc, vc, ks, vs, n), dict(out=(torch.empty(1, 2, 8, 64, device="cuda"), None))),
                     ((kc, vc, ks, vs, n), dict(out=(torch.empty(1, 2, 7, 64, device="cuda"),) * 2)),
                     ((kc, vc, ks, vs, n), dict(out=(torch.empty(1, 2, 8, 64, device="cuda"),) * 2)),
                     ((kc, vc, ks, vs, n), dict(dtype="bf16"))):
        with pytest.raises((RuntimeError, TypeError)):
            fc.dequantize_cache(*args, **kw)
    e = torch.empty(1, 2, 0, 64, dtype=I8, device="cuda")
    s = torch.empty(1, 2, 0, device="cuda")
    assert fc.dequantize_cache(e, e, s, s, n)[0].shape == (1, 2, 0, 64)


def test_in_a_graph_and_versions(gpu_device):
    """Append and read-back captured together replay as the cache grows; what is written in place counts as written."""
    kc, vc, ks, vs = caches(1, 2, 2, 64, 64, F8)
    x = draw(1, 2, 2, 3, 64, FH)
    f, _ = rot.rotary_frequencies(64, device="cuda")
    n = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    versions = [t._version for t in (kc, vc, ks, vs)]
    fc.quantized_append(x, x, x, kc, vc, ks, vs, n, f)
    assert all(t._version > v for t, v in zip((kc, vc, ks, vs), versions))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fc.quantized_append(x, x, x, kc, vc, ks, vs, n, f)
        n += 3
        out = fc.dequantize_cache(kc, vc, ks, vs, n, dtype=FH)
    n.copy_(torch.tensor([0, 5], dtype=torch.int32))
    mine = [t.clone() for t in (kc, vc, ks, vs, n)]
    for turn in range(4):
        x.copy_(draw(10 + turn, 2, 2, 3, 64, FH))
        graph.replay()
        torch.cuda.synchronize()
        want = fc.quantized_append(x, x, x, *mine, f)
        mine[4] += 3
        back = fc.dequantize_cache(*mine, dtype=FH)
        assert torch.equal(y, want) and torch.equal(n, mine[4])
        assert torch.equal(out[0], back[0]) and torch.equal(out[1], back[1])


def nearest(y, s, code, kind):
    """How far codes are from being the nearest of y / s (float64), in half steps."""
    t, c = y / s[..., None], code.float().double()
    if kind == I8:
        return ((t - c).abs() / 0.5).max().item()
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)  # of e4m3 where t is
    return ((t - c).abs() / (step / 2)).max().item()


@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("dtype", [BF, FH, FS])
def test_codes_at_borders(gpu_device, kind, dtype):
    """Values are divided by their scale exactly, ties go to the even code; keys are off by far less than 32 bits are.

    e4m3 is rounded from a quotient of 32 bits, 2^-24 of at most 32 half steps off: 2^-19 of a half step.  64 bits leave 1e-11 of a row's largest size (positions up to 3e5 times 2^-53 and the series' 4e-13), 448 and 127 times
    that on the codes' scale, against half steps of at least 2^-10 and 2^-1."""
    B, H, S, D = 2, 4, 500, 128
    k, v = draw(1, B, H, S, D, dtype), draw(2, B, H, S, D, dtype)
    v[0, :, ::3] = (v[0, :, ::3] * 64).round().clamp(-126, 126) / 2  # whole halves
    v[0, :, ::3, 5] = 127.0 if kind == I8 else 448.0  # and a scale of 1
    v[1, :, ::5, 7] = 254.0 if kind == I8 else 28.0   # or 2, or 1/16
    kc, vc, ks, vs = caches(3, B, H, S, D, kind)
    f, w = rot.rotary_frequencies(D, device="cuda")[0], weight(4, D, dtype)
    pos = (torch.arange(S) * 601 % 300000).expand(B, S).contiguous()
    fc.quantized_append(k[:, :0], k, v, kc, vc, ks, vs, torch.zeros(B, dtype=torch.int32, device="cuda"), f,
                        positions=pos.cuda(), query_weight=w, key_weight=w, eps=1e-4)
    x = v.double()
    s = (x.abs().amax(dim=-1).clamp(min=2.0 ** -100) / orc.TOP[kind]).float()
    t = (x / s.double()[..., None])
    want = t.round().to(I8) if kind == I8 else None
    assert torch.equal(vs, s) and (want is None or torch.equal(vc, want))
    once = 2.0 ** -19 if kind == F8 else 0.0
    assert nearest(x, s.double(), vc, kind) <= 1.0 + once
    if kind == F8:  # a tie's code is even
        tie = (t - vc.float().double()).abs() * 2 == torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
        assert int(tie.sum()) > 100 and bool((bits(vc)[tie] % 2 == 0).all())
    y, _ = orc.norm_rotary(k.cpu().double(), w.cpu().double(), f.cpu(), pos, False, 1.0, float(torch.tensor(1e-4)))
    size = y.abs().amax(dim=-1) / orc.TOP[kind]
    assert bool(((ks.cpu().double() - size).abs() <= size * (2.0 ** -24 + 2e-11)).all())
    assert nearest(y, ks.cpu().double(), kc.cpu(), kind) <= 1.0 + once + 1e-11 * (448 * 2 ** 10 if kind == F8 else 127 * 2)
