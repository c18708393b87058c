"""Tree attention over a cache of 8 bits on the GPU against the float64 oracle, element by element with the tolerance that
follows from the kernel's arithmetic (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_quant_cache import bits
from test_gpu_tree import check, draw, tree

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
F8, I8 = torch.float8_e4m3fn, torch.int8


def cache(seed, B, H, C, D, kind, spread=0.3):
    """Codes and scales of rows that differ in size."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, C, D, generator=g) * torch.exp(spread * torch.randn(B, H, C, 1, generator=g))
    s = (x.abs().amax(dim=-1) / orc.TOP[kind]).float()
    y = x / s[..., None]
    return (y.round().to(I8) if kind == I8 else y.to(F8)).cuda(), s.cuda()


CASES = [
    # dtype, cache, B, Hq, Hkv, T, C, D, lengths, mask, window, cap, layout
    (BF, F8, 2, 8, 2, 1, 300, 128, [299, 0], None, 0, 0.0, "bnsd"),
    (BF, I8, 3, 8, 2, 8, 700, 128, [692, 1, 333], "shared", 0, 0.0, "bsnd"),
    (FH, F8, 2, 7, 1, 13, 4097, 64, [4084, 2049], "batch", 0, 30.0, "bnsd"),
    (FH, I8, 1, 4, 4, 64, 130, 64, [66], "shared", 0, 0.0, "bnsd"),
    (BF, F8, 2, 4, 2, 33, 900, 256, [800, 31], "batch", 200, 50.0, "bsnd"),
    (FH, I8, 1, 4, 2, 9, 2000, 256, [1991], None, 5, 0.0, "bnsd"),
    (FH, F8, 2, 3, 1, 5, 64, 32, [59, 32], "holes", 0, 0.0, "bnsd"),
    (BF, I8, 2, 2, 2, 40, 40, 32, [0, 0], "holes", 0, 0.0, "bnsd"),      # nothing cached: rows without keys
    (BF, F8, 1, 2, 1, 100, 1000, 64, [500], "holes", 3, 0.0, "bnsd"),    # a window shorter than the tree
    (BF, F8, 1, 32, 8, 2, 9000, 128, [8998], None, 0, 0.0, "bnsd"),      # many splits
    (FH, I8, 4, 2, 1, 1, 20000, 128, [19999, 3, 0, 7777], None, 0, 0.0, "bnsd"),  # unequal lengths, many splits
    (FH, F8, 1, 1, 1, 300, 1200, 64, [900], "shared", 0, 0.0, "bnsd"),   # more drafted tokens than a tile
    (BF, I8, 1, 8, 2, 30, 1500, 128, [1470], "batch", 0, 0.0, "bnsd"),   # pairs of row tiles, an odd one
    (FH, F8, 2, 7, 1, 64, 800, 128, [700, 3], "holes", 50, 30.0, "bsnd"),
    (BF, F8, 3, 5, 1, 13, 300, 128, [287, 1, 100], None, 20, 0.0, "bsnd"),
    (FH, I8, 1, 9, 1, 20, 2000, 32, [1980], "shared", 0, 0.0, "bnsd"),
    (BF, I8, 1, 8, 1, 40, 600, 256, [560], "shared", 0, 0.0, "bnsd"),
    (BF, F8, 1, 1, 1, 1, 1, 64, [0], None, 0, 0.0, "bnsd"),              # a token alone
]


def run_case(i):
    dtype, kind, B, Hq, Hkv, T, C, D, n, mask, window, cap, layout = CASES[i]
    q = draw(i, B, Hq, T, D, dtype, layout)
    (kc, ks), (vc, vs) = cache(50 + i, B, Hkv, C, D, kind), cache(90 + i, B, Hkv, C, D, kind, 1.0)
    m = depths = None
    if mask:
        made = [tree(T, 7 * i + b, mask) for b in range(B if mask in ("batch", "holes") else 1)]
        m = torch.stack([x for x, _ in made])
        depths = torch.stack([d for _, d in made]).expand(B, T)
    kw = dict(sliding_window=window, soft_cap=cap, scale=0.11 if cap else None)
    return q, kc, vc, ks, vs, torch.tensor(n, dtype=torch.int32), m, depths, kw, dtype


def of_case(i):
    q, kc, vc, ks, vs, n, m, depths, kw, dtype = run_case(i)
    if m is not None:
        kw = dict(kw, tree_mask=m.cuda(), depths=depths.cuda())
    return (q, kc, vc, ks, vs, n.cuda()), kw


@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_oracle(gpu_device, i):
    q, kc, vc, ks, vs, n, m, depths, kw, dtype = run_case(i)
    args, gpu = of_case(i)
    o, lse = fc.quantized_tree_attention(*args, return_lse=True, **gpu)
    assert o.shape == q.shape and o.dtype == dtype and lse.shape == q.shape[:3] and lse.dtype == FS
    ro, rl, to, tl = orc.quantized_tree_attention(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), n, m,
                                                  kw["sliding_window"], depths, kw["scale"], kw["soft_cap"], dtype)
    check("o", o, ro, to)
    check("lse", lse, rl, tl)
    assert torch.equal(o, fc.quantized_tree_attention(*args, **gpu))


def test_negative_and_no_scale(gpu_device):
    (q, kc, vc, ks, vs, n), _ = of_case(1)
    for scale in (-0.07, 0.0):
        o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, scale=scale, return_lse=True)
        ro, rl, to, tl = orc.quantized_tree_attention(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), n.cpu(), scale=scale)
        check("o", o, ro, to)
        check("lse", lse, rl, tl)


@pytest.mark.parametrize("kind", [F8, I8])
def test_scales_of_any_size(gpu_device, kind):
    """fp16: values of 1e-6 to 1e6, no value's scale, scales that grow and shrink along the cache."""
    q = draw(1, 1, 4, 2, 64, FH)
    (kc, ks), (vc, vs) = cache(2, 1, 2, 700, 64, kind), cache(3, 1, 2, 700, 64, kind)
    n = torch.tensor([698], dtype=torch.int32)
    for f in (torch.full((700,), 1e-6), torch.full((700,), 100.0), torch.zeros(700), torch.logspace(-6, 2, 700),
              torch.logspace(2, -6, 700)):
        s = vs * f.cuda()
        o, lse = fc.quantized_tree_attention(q, kc, vc, ks, s, n.cuda(), return_lse=True)
        ro, rl, to, tl = orc.quantized_tree_attention(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), s.cpu(), n, dtype=FH)
        check("o", o, ro, to)
        check("lse", lse, rl, tl)


def test_what_the_cache_holds_behind_does_not_matter(gpu_device):
    """NaN behind lengths + T, and in keys that no token sees, leave the results as they are."""
    (q, kc, vc, ks, vs, n), kw = of_case(2)
    a = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    for b, x in enumerate(n.tolist()):
        bits(kc)[b, :, x + 13:] = 0x7f
        bits(vc)[b, :, x + 13:] = 0xff
        ks[b, :, x + 13:] = float("nan")
        vs[b, :, x + 13:] = float("inf")
    c = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    m = kw["tree_mask"]
    m[:, :, 12] = False  # the last token's key: seen by nobody, and not a number
    m[:, 12, 11] = True
    d = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    for b, x in enumerate(n.tolist()):
        ks[b, :, x + 12] = float("nan")
    e = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    assert torch.equal(d[0], e[0]) and torch.equal(d[1], e[1])


def test_a_row_that_is_not_a_number(gpu_device):
    """A key whose scale is NaN makes NaN of the tokens that see it; a query row of NaN of itself alone."""
    (q, kc, vc, ks, vs, n), _ = of_case(0)
    good = fc.quantized_tree_attention(q, kc, vc, ks, vs, n)
    q2 = q.clone()
    q2[0, 3, 0, 5] = float("nan")
    o = fc.quantized_tree_attention(q2, kc, vc, ks, vs, n)
    assert bool(torch.isnan(o[0, 3]).all())
    o[0, 3] = good[0, 3]
    assert torch.equal(o, good)
    ks[0, 1, 17] = float("nan")
    o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True)
    assert bool(torch.isnan(o[0, 4:]).all()) and bool(torch.isnan(lse[0, 4:]).all())
    assert torch.equal(o[0, :4], good[0, :4]) and torch.equal(o[1], good[1])


def test_lengths_that_do_not_fit(gpu_device):
    (q, kc, vc, ks, vs, n), kw = of_case(1)
    n2 = torch.tensor([693, -1, 333], dtype=torch.int32, device="cuda")
    good = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, n2, return_lse=True, **kw)
    assert bool(torch.isnan(o[:2]).all()) and bool(torch.isnan(lse[:2]).all())
    assert torch.equal(o[2], good[0][2]) and torch.equal(lse[2], good[1][2])


def test_strides_streams_and_graphs(gpu_device):
    """A cache of heads innermost, keys and values in one buffer; another stream; a graph replayed as the lengths grow."""
    (q, kc, vc, ks, vs, n), kw = of_case(3)
    want = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    both = torch.stack((bits(kc), bits(vc)), dim=3).transpose(1, 2).contiguous()  # [B, C, H, 2, D]
    k2, v2 = (both[:, :, :, j].transpose(1, 2).view(I8) for j in range(2))
    got = fc.quantized_tree_attention(q, k2, v2, ks, vs, n, return_lse=True, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(*kc.shape[:3], 65, dtype=I8, device="cuda")
    odd[..., 1:] = kc
    got = fc.quantized_tree_attention(q, odd[..., 1:], vc, ks, vs, n, return_lse=True, **kw)  # copied by the call
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0])
    (q, kc, vc, ks, vs, n), kw = of_case(10)
    graph = torch.cuda.CUDAGraph()
    fc.quantized_tree_attention(q, kc, vc, ks, vs, n)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True)
    for lengths in ([1, 2, 3, 4], [19999, 0, 19999, 19999], [0, 0, 0, 0], [400, 19999, 31, 33]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = fc.quantized_tree_attention(q, kc, vc, ks, vs, n, return_lse=True)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_empty_and_refused(gpu_device):
    (q, kc, vc, ks, vs, n), _ = of_case(0)
    o, lse = fc.quantized_tree_attention(q[:, :, :0], kc, vc, ks, vs, n, return_lse=True)
    assert o.shape == (2, 8, 0, 128) and lse.shape == (2, 8, 0)
    ok = dict(query=q, key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, lengths=n)
    for kw in (dict(query=q.float()), dict(key_cache=q), dict(value_cache=bits(vc)), dict(key_scales=ks[:1]),
               dict(value_scales=vs.half()), dict(key_scales=ks.cpu()), dict(lengths=n.long()), dict(soft_cap=float("nan")),
               dict(query=q.clone().requires_grad_()), dict(key_scales=ks.clone().requires_grad_()),
               dict(tree_mask=torch.ones(2, 2, device="cuda", dtype=torch.bool)),
               dict(query=q.expand(2, 8, 1, 128).repeat(1, 1, 301, 1))):
        with pytest.raises(RuntimeError):
            fc.quantized_tree_attention(**dict(ok, **kw))
    with pytest.raises(AssertionError):
        fc.quantized_tree_attention(**dict(ok, query=q[:, :7]))
    with pytest.raises(AssertionError):
        fc.quantized_tree_attention(**dict(ok, query=q[..., :64].contiguous()))


UNEVEN = [
    # dtype, cache, B, Hq, Hkv, T, C, D, lengths, window
    (BF, F8, 2, 16, 8, 256, 20300, 64, [20000, 12000], 0),      # workgroups whose share ends in the next head's tiles
    (FH, I8, 3, 8, 8, 200, 9000, 128, [8800, 4100, 6400], 0),
    (BF, I8, 4, 8, 4, 160, 9000, 64, [8840, -1, 4500, 8840], 0),  # one that does not fit among them
    (FH, F8, 3, 8, 4, 250, 20000, 128, [19000, 2000, 5000], 9000),
    (BF, F8, 9, 16, 4, 16, 9000, 128, [8000, 8100, 0, 8984, 5000, 5100, 33, 1, 7000], 0),
]


@pytest.mark.parametrize("i", range(len(UNEVEN)))
def test_sequences_of_uneven_lengths(gpu_device, i):
    dtype, kind, B, Hq, Hkv, T, C, D, n, window = UNEVEN[i]
    q = draw(i, B, Hq, T, D, dtype)
    (kc, ks), (vc, vs) = cache(50 + i, B, Hkv, C, D, kind), cache(90 + i, B, Hkv, C, D, kind, 1.0)
    lengths = torch.tensor(n, dtype=torch.int32)
    args = (q, kc, vc, ks, vs, lengths.cuda())
    o, lse = fc.quantized_tree_attention(*args, sliding_window=window, return_lse=True)
    fits = lengths >= 0
    for b in range(B):
        if not fits[b]:
            assert bool(o[b].isnan().all()) and bool(lse[b].isnan().all())
            continue
        ro, rl, to, tl = orc.quantized_tree_attention(*(x[b:b + 1].cpu() for x in args), window=window, dtype=dtype)
        check("o", o[b:b + 1], ro, to)
        check("lse", lse[b:b + 1], rl, tl)
    again = fc.quantized_tree_attention(*args, sliding_window=window, return_lse=True)
    assert torch.equal(o[fits.cuda()], again[0][fits.cuda()]) and torch.equal(lse[fits.cuda()], again[1][fits.cuda()])
