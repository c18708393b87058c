"""Tree attention on the GPU against the float64 oracle, element by element with the tolerance that follows from the
kernel's arithmetic (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
import npu_flash_attention as nfa
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def tree(T, seed, kind="tree"):
    """[T, T] bool and depths: a random tree, or a mask with empty rows."""
    g = torch.Generator().manual_seed(seed)
    m, d = torch.zeros(T, T, dtype=torch.bool), []
    for t in range(T):
        parent = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
        if parent >= 0:
            m[t] = m[parent]
        m[t, t] = True
        d.append(d[parent] + 1 if parent >= 0 else 0)
    if kind == "holes":
        m[::3] = False  # tokens that see none of the tree, not even themselves
    return m, torch.tensor(d, dtype=torch.int32)


def draw(seed, B, H, S, D, dtype, layout="bnsd", spread=1.0):
    g = torch.Generator().manual_seed(seed)
    if layout == "bsnd":
        return (torch.randn(B, S, H, D, generator=g) * spread).to(dtype).cuda().transpose(1, 2)
    return (torch.randn(B, H, S, D, generator=g) * spread).to(dtype).cuda()


def check(name, x, ref, tol):
    x = x.cpu().double()
    assert torch.equal(torch.isnan(x), torch.isnan(ref)), f"{name}: NaN where none is due, or none where it is"
    fin = torch.isfinite(ref)
    assert torch.equal(x[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), f"{name}: infinities differ"
    worst = ((x[fin] - ref[fin]).abs() / tol[fin]).max().item() if bool(fin.any()) else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} tolerances"


CASES = [
    # dtype, B, Hq, Hkv, T, C, D, lengths, mask, window, cap, layout
    (BF, 2, 8, 2, 1, 300, 128, [299, 0], None, 0, 0.0, "bnsd"),
    (BF, 3, 8, 2, 8, 700, 128, [692, 1, 333], "shared", 0, 0.0, "bsnd"),
    (FH, 2, 7, 1, 13, 4097, 64, [4084, 2049], "batch", 0, 30.0, "bnsd"),
    (FH, 1, 4, 4, 64, 130, 64, [66], "shared", 0, 0.0, "bnsd"),
    (BF, 2, 4, 2, 33, 900, 256, [800, 31], "batch", 200, 50.0, "bsnd"),
    (BF, 1, 4, 2, 9, 2000, 256, [1991], None, 5, 0.0, "bnsd"),
    (FH, 2, 3, 1, 5, 64, 32, [59, 32], "holes", 0, 0.0, "bnsd"),
    (BF, 2, 2, 2, 40, 40, 32, [0, 0], "holes", 0, 0.0, "bnsd"),      # nothing cached: rows without keys
    (BF, 1, 2, 1, 100, 1000, 64, [500], "holes", 3, 0.0, "bnsd"),    # a window shorter than the tree
    (FS, 2, 4, 2, 6, 500, 128, [494, 100], "shared", 0, 0.0, "bsnd"),
    (FS, 1, 2, 1, 17, 3000, 64, [2900], "batch", 0, 30.0, "bnsd"),
    (FS, 1, 2, 2, 3, 90, 256, [87], None, 40, 0.0, "bnsd"),
    (FS, 1, 3, 1, 2, 70, 32, [68], None, 0, 0.0, "bnsd"),
    (BF, 1, 32, 8, 2, 9000, 128, [8998], None, 0, 0.0, "bnsd"),      # many splits
    (BF, 4, 2, 1, 1, 20000, 128, [19999, 3, 0, 7777], None, 0, 0.0, "bnsd"),  # unequal lengths, many splits
    (FH, 1, 1, 1, 300, 1200, 64, [900], "shared", 0, 0.0, "bnsd"),   # more drafted tokens than a tile
    # several row tiles, whose waves share key tiles: full fours, padded ones, pairs; more waves than key tiles
    (BF, 1, 8, 2, 30, 1500, 128, [1470], "batch", 0, 0.0, "bnsd"),
    (FH, 2, 7, 1, 64, 800, 128, [700, 3], "holes", 50, 30.0, "bsnd"),
    (BF, 2, 6, 1, 27, 600, 128, [500, 0], "shared", 0, 0.0, "bnsd"),
    (BF, 3, 5, 1, 13, 300, 128, [287, 1, 100], None, 20, 0.0, "bsnd"),
    (FH, 1, 9, 1, 20, 2000, 32, [1980], "shared", 0, 0.0, "bnsd"),
    (BF, 2, 8, 1, 40, 60, 64, [20, 0], "batch", 7, 0.0, "bnsd"),
    (BF, 1, 4, 1, 70, 9000, 128, [8930], "shared", 0, 0.0, "bsnd"),
]


def run_case(i, **over):
    dtype, B, Hq, Hkv, T, C, D, n, mask, window, cap, layout = CASES[i]
    q, kc, vc = draw(i, B, Hq, T, D, dtype, layout), draw(50 + i, B, Hkv, C, D, dtype, layout), \
        draw(90 + i, B, Hkv, C, D, dtype, layout)
    m = depths = None
    if mask:
        made = [tree(T, 7 * i + b, mask) for b in range(B if mask in ("batch", "holes") else 1)]
        m = torch.stack([x for x, _ in made])
        depths = torch.stack([d for _, d in made]).expand(B, T)
    kw = dict(sliding_window=window, soft_cap=cap, scale=0.11 if cap else None)
    return q, kc, vc, torch.tensor(n, dtype=torch.int32), m, depths, kw, dtype


def to_oracle(q, kc, vc, n, m, depths, kw, dtype):
    return orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), n, m, kw["sliding_window"], depths, kw["scale"],
                              kw["soft_cap"], dtype)


@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_oracle(gpu_device, i):
    q, kc, vc, n, m, depths, kw, dtype = run_case(i)
    if m is not None:
        kw = dict(kw, tree_mask=m.cuda(), depths=depths.cuda())
    o, lse = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True, **kw)
    assert o.shape == q.shape and o.dtype == dtype and lse.shape == q.shape[:3] and lse.dtype == FS
    kw.pop("tree_mask", None), kw.pop("depths", None)
    ro, rl, to, tl = to_oracle(q, kc, vc, n, m, depths, kw, dtype)
    check("o", o, ro, to)
    check("lse", lse, rl, tl)
    again = fc.tree_attention(q, kc, vc, n.cuda(), None if m is None else m.cuda(),
                              depths=None if depths is None else depths.cuda(), **kw)
    assert torch.equal(o, again)


def test_what_the_cache_holds_behind_does_not_matter(gpu_device):
    """NaN and infinities behind lengths + T, and in keys that no token sees, leave the results as they are."""
    q, kc, vc, n, m, depths, kw, dtype = run_case(2)
    a = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True, **kw)
    for b, x in enumerate(n.tolist()):
        kc[b, :, x + 13:] = float("nan")
        vc[b, :, x + 13:] = float("inf")
    c = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True, **kw)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    m[:, :, 12] = False  # the last token's key: seen by nobody, and not a number
    m[:, 12, 11] = True
    d = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True, **kw)
    for b, x in enumerate(n.tolist()):
        kc[b, :, x + 12] = float("nan")
    e = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True, **kw)
    assert torch.equal(d[0], e[0]) and torch.equal(d[1], e[1])


@pytest.mark.parametrize("dtype", [BF, FS])
def test_nan_scores_and_sequences_that_do_not_fit(gpu_device, dtype):
    q, kc, vc = draw(1, 4, 2, 3, 64, dtype), draw(2, 4, 1, 200, 64, dtype), draw(3, 4, 1, 200, 64, dtype)
    n = torch.tensor([197, 198, -1, 2147483647], dtype=torch.int32)  # the first alone fits
    o, lse = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True)
    ref = orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), n, dtype=dtype)
    check("o", o, ref[0], ref[2])
    check("lse", lse, ref[1], ref[3])
    kc[0, 0, 50, 3] = float("nan")  # a cached key every row sees
    q[0, 1, 2, 5] = float("nan")
    o, lse = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True)
    assert bool(torch.isnan(o).all()) and bool(torch.isnan(lse).all())


def test_decoding_agrees_with_the_forward(gpu_device):
    """One token per sequence over a cache filled to its end is the forward over it."""
    q, kc, vc = draw(1, 2, 8, 1, 128, BF), draw(2, 2, 2, 1000, 128, BF), draw(3, 2, 2, 1000, 128, BF)
    o, lse = fc.tree_attention(q, kc, vc, torch.tensor([999, 999], dtype=torch.int32, device="cuda"), return_lse=True)
    fo, fl = nfa.npu_flash_attention_forward(q, kc, vc, return_lse=True)
    ref = orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), [999, 999], dtype=BF)
    check("o", o, ref[0], ref[2])
    check("the forward's o", fo, ref[0], ref[2])
    check("lse", lse, fl.cpu().double(), 2 * ref[3])


def test_layouts_negative_scale_and_offsets_past_32_bits(gpu_device):
    q, kc, vc, n, m, depths, kw, dtype = run_case(1)
    base = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), scale=-0.07)
    ref = orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), n, m, scale=-0.07, dtype=dtype)
    check("o", base, ref[0], ref[2])
    both = torch.stack((kc.transpose(1, 2), vc.transpose(1, 2)), dim=2)  # [B, C, 2, H, D]
    x = fc.tree_attention(q.contiguous(), both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), n.cuda(),
                          m[0].cuda().long(), scale=-0.07)
    assert torch.equal(base, x)
    # one head of a cache whose rows lie 2^22 elements apart: row 520 starts past 2^31
    wide = torch.zeros(600 << 22, dtype=dtype, device="cuda")[:600 * (1 << 22)].view(1, 600, 1 << 22)
    k2, v2 = draw(5, 1, 1, 600, 128, dtype), draw(6, 1, 1, 600, 128, dtype)
    wide[0, :, :128], wide[0, :, 128:256] = k2[0, 0], v2[0, 0]
    q2, n2 = draw(7, 1, 4, 2, 128, dtype), torch.tensor([598], dtype=torch.int32, device="cuda")
    assert torch.equal(fc.tree_attention(q2, wide[None, :, :, :128], wide[None, :, :, 128:256], n2),
                       fc.tree_attention(q2, k2, v2, n2))


def test_refusals(gpu_device):
    q, c = draw(1, 2, 4, 3, 64, BF), draw(2, 2, 2, 20, 64, BF)
    n = torch.tensor([4, 5], dtype=torch.int32, device="cuda")
    m = torch.ones(3, 3, dtype=torch.bool, device="cuda")
    bad = [dict(lengths=n.cpu()), dict(lengths=n.long()), dict(tree_mask=m.cpu()), dict(tree_mask=m[:2]),
           dict(tree_mask=m.float()), dict(tree_mask=m, sliding_window=4),
           dict(sliding_window=4, depths=torch.zeros(3, device="cuda")),
           dict(sliding_window=4, depths=torch.zeros(4, dtype=torch.int32, device="cuda")),
           dict(query=q.half()), dict(query=q.clone().requires_grad_()), dict(query=q[0]), dict(scale=float("nan"))]
    for kw in bad:
        args = dict(query=q, key_cache=c, value_cache=c, lengths=n)
        args.update(kw)
        with pytest.raises(RuntimeError):
            fc.tree_attention(**args)
    with pytest.raises(RuntimeError, match="fit"):
        fc.tree_attention(draw(1, 2, 4, 21, 64, BF), c, c, n)
    with pytest.raises(AssertionError):
        fc.tree_attention(draw(1, 2, 3, 3, 64, BF), c, c, n)
    with pytest.raises(AssertionError):
        fc.tree_attention(q[:1], c, c, n)
    o, lse = fc.tree_attention(q[:, :, :0], c, c, n, return_lse=True)
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    assert fc.tree_attention(q.clone().requires_grad_().detach(), c, c, n).shape == q.shape


def test_graph_replays_as_the_cache_grows(gpu_device):
    """Captured with one set of lengths, replayed with others: the plan follows the lengths on the device.  A second
    graph with a workspace of its own runs between."""
    B, Hq, Hkv, T, C, D = 2, 8, 2, 4, 9000, 128
    q, kc, vc = draw(1, B, Hq, T, D, BF), draw(2, B, Hkv, C, D, BF), draw(3, B, Hkv, C, D, BF)
    n = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fc.tree_attention(q, kc, vc, n)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = fc.tree_attention(q, kc, vc, n)
    with torch.cuda.graph(g2):
        o2 = fc.tree_attention(q, kc, vc, n, scale=0.2)
    for a, b in ((8996, 17), (0, 8000), (4000, 4000)):
        n.copy_(torch.tensor([a, b], dtype=torch.int32))
        e1, e2 = fc.tree_attention(q, kc, vc, n), fc.tree_attention(q, kc, vc, n, scale=0.2)
        torch.cuda.synchronize()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, e1) and torch.equal(o2, e2)


@pytest.mark.parametrize("dtype,T,D,window", [(BF, 1, 32, 0), (FH, 3, 128, 90), (FS, 2, 64, 0)])
def test_many_sequences_of_unequal_lengths(gpu_device, dtype, T, D, window):
    """More sequences than a wave has lanes, from nothing cached to a full cache, one that does not fit among them."""
    B, C = 150, 700
    g = torch.Generator().manual_seed(5)
    n = torch.randint(0, C - T + 1, (B,), generator=g).int()
    n[::7], n[3::11], n[70] = 0, C - T, C
    q, kc, vc = draw(1, B, 2, T, D, dtype), draw(2, B, 1, C, D, dtype, "bsnd"), draw(3, B, 1, C, D, dtype)
    o, lse = fc.tree_attention(q, kc, vc, n.cuda(), sliding_window=window, return_lse=True)
    ref = orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), n, None, window, dtype=dtype)
    check("o", o, ref[0], ref[2])
    check("lse", lse, ref[1], ref[3])


def test_caches_of_one_row_and_strides_of_size_one_dimensions(gpu_device):
    q, k, v = draw(1, 3, 4, 1, 64, BF), draw(2, 3, 2, 1, 64, BF), draw(3, 3, 2, 1, 64, BF)
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    o, lse = fc.tree_attention(q, k, v, n, return_lse=True)
    ref = orc.tree_attention(q.cpu(), k.cpu(), v.cpu(), n.cpu(), dtype=BF)
    check("o", o, ref[0], ref[2])
    check("lse", lse, ref[1], ref[3])
    far = torch.as_strided(k, k.shape, (128, 64, 1 << 40, 1))  # no second row lies there
    assert torch.equal(o, fc.tree_attention(q, far, v, n))
    assert torch.equal(o, fc.tree_attention(torch.as_strided(q, q.shape, (256, 64, 3, 1)), k, v, n))


def test_what_a_workspace_holds_does_not_matter(gpu_device):
    q, kc, vc, n, m, depths, kw, dtype = run_case(13)
    a = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True, **kw)
    torch.cuda.synchronize()
    for fill in (float("nan"), float("inf")):
        junk = [torch.full((1 << s,), fill, device="cuda") for s in range(14, 23)]
        del junk  # what the allocator hands out next
        b = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_streams_at_once(gpu_device):
    q, kc, vc, n, m, depths, kw, dtype = run_case(13)
    n = n.cuda()
    want = [fc.tree_attention(q, kc, vc, n, scale=s) for s in (0.05, 0.2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fc.tree_attention(q, kc, vc, n, scale=(0.05, 0.2)[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_more_drafted_tokens_than_workgroups_at_once(gpu_device):
    """A chain of 2000 tokens behind 900 cached ones: its row tiles alone fill the chip, each takes all keys."""
    q, kc, vc = draw(1, 1, 8, 2000, 32, FH), draw(2, 1, 1, 3000, 32, FH), draw(3, 1, 1, 3000, 32, FH)
    n = torch.tensor([900], dtype=torch.int32)
    o, lse = fc.tree_attention(q, kc, vc, n.cuda(), return_lse=True)
    ref = orc.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), n, dtype=FH)
    check("o", o, ref[0], ref[2])
    check("lse", lse, ref[1], ref[3])


def test_a_row_that_is_not_a_number_stays_alone(gpu_device):
    q, kc, vc, n, m, depths, kw, dtype = run_case(1)
    a = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True)
    q[1, 3, 5, 7] = float("nan")
    b = fc.tree_attention(q, kc, vc, n.cuda(), m.cuda(), return_lse=True)
    assert bool(torch.isnan(b[0][1, 3, 5]).all()) and bool(torch.isnan(b[1][1, 3, 5]))
    b[0][1, 3, 5], b[1][1, 3, 5] = a[0][1, 3, 5], a[1][1, 3, 5]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
