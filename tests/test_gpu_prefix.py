"""Attention of sequences behind a shared prefix on the GPU against the float64 oracle, element by element with the
tolerance that follows from the kernel's arithmetic (oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_tree import check, draw, tree

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # dtype, B, Hq, Hkv, T, P, C, D, lengths, mask, window, cap, layout
    (BF, 2, 8, 2, 1, 300, 40, 128, [39, 0], None, 0, 0.0, "bnsd"),
    (BF, 3, 8, 2, 8, 700, 333, 128, [300, 1, 0], "shared", 0, 0.0, "bsnd"),
    (FH, 2, 7, 1, 13, 4097, 130, 64, [117, 64], "batch", 0, 30.0, "bnsd"),
    (FH, 1, 4, 4, 64, 130, 70, 64, [6], "shared", 0, 0.0, "bnsd"),
    (BF, 2, 4, 2, 33, 900, 300, 256, [200, 31], "batch", 500, 50.0, "bsnd"),
    (BF, 3, 4, 2, 9, 2000, 40, 256, [31, 3, 0], None, 25, 0.0, "bnsd"),   # a window that ends in the prefix, or behind it
    (FH, 2, 3, 1, 5, 64, 64, 32, [59, 32], "holes", 0, 0.0, "bnsd"),
    (BF, 2, 2, 2, 40, 33, 40, 32, [0, 0], "holes", 3, 0.0, "bnsd"),       # rows without keys
    (FS, 2, 4, 2, 6, 500, 106, 128, [100, 7], "shared", 0, 0.0, "bsnd"),
    (FS, 1, 2, 1, 17, 3000, 90, 64, [50], "batch", 0, 30.0, "bnsd"),
    (FS, 5, 2, 2, 3, 90, 20, 256, [17, 0, 3, 9, 16], None, 40, 0.0, "bnsd"),
    (FS, 1, 3, 1, 2, 1, 2, 32, [0], None, 0, 0.0, "bnsd"),
    (BF, 40, 8, 2, 1, 1000, 50, 128, list(range(40)), None, 0, 0.0, "bnsd"),  # many sequences: several row tiles
    (FH, 70, 4, 1, 2, 513, 40, 64, [i % 38 for i in range(70)], "shared", 0, 0.0, "bsnd"),
    (BF, 9, 7, 1, 4, 5000, 300, 128, [296, 0, 100, 1, 2, 3, 250, 31, 32], "batch", 0, 20.0, "bnsd"),
    (FH, 33, 8, 8, 1, 200, 9, 32, [i % 9 for i in range(33)], None, 0, 0.0, "bnsd"),
    (BF, 17, 8, 4, 3, 257, 64, 256, [i for i in range(17)], "shared", 270, 0.0, "bnsd"),
    (BF, 1, 1, 1, 1, 1, 1, 64, [0], None, 0, 0.0, "bnsd"),
    (FH, 130, 16, 2, 1, 2049, 33, 128, [i % 33 for i in range(130)], None, 0, 0.0, "bnsd"),
    (BF, 64, 8, 1, 2, 1500, 20, 64, [i % 19 for i in range(64)], "batch", 700, 0.0, "bnsd"),
]


def run_case(i):
    dtype, B, Hq, Hkv, T, P, C, D, n, mask, window, cap, layout = CASES[i]
    q, kc, vc = draw(i, B, Hq, T, D, dtype, layout), draw(50 + i, B, Hkv, C, D, dtype, layout), \
        draw(90 + i, B, Hkv, C, D, dtype, layout)
    pk, pv = draw(130 + i, 1, Hkv, P, D, dtype, layout)[0], draw(170 + i, 1, Hkv, P, D, dtype)[0]
    m = depths = None
    if mask:
        made = [tree(T, 7 * i + b, mask) for b in range(B if mask in ("batch", "holes") else 1)]
        m = torch.stack([x for x, _ in made])
        depths = torch.stack([d for _, d in made]).expand(B, T)
    kw = dict(sliding_window=window, soft_cap=cap, scale=0.11 if cap else None)
    return q, pk, pv, kc, vc, torch.tensor(n, dtype=torch.int32), m, depths, kw, dtype


def of_case(i):
    q, pk, pv, kc, vc, n, m, depths, kw, dtype = run_case(i)
    if m is not None:
        kw = dict(kw, tree_mask=m.cuda(), depths=depths.cuda())
    return (q, pk, pv, kc, vc, n.cuda()), kw


def oracle(q, pk, pv, kc, vc, n, m, depths, kw, dtype):
    return orc.prefix_attention(*(x.cpu() for x in (q, pk, pv, kc, vc)), n, m, kw["sliding_window"], depths, kw["scale"],
                                kw["soft_cap"], dtype)


@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_oracle(gpu_device, i):
    case = run_case(i)
    args, kw = of_case(i)
    o, lse = fc.shared_prefix_attention(*args, return_lse=True, **kw)
    assert o.shape == args[0].shape and o.dtype == args[0].dtype and lse.shape == o.shape[:3] and lse.dtype == FS
    ro, rl, to, tl = oracle(*case)
    check("o", o, ro, to)
    check("lse", lse, rl, tl)
    assert torch.equal(o, fc.shared_prefix_attention(*args, **kw))


def test_no_prefix_is_tree_attention(gpu_device):
    (q, pk, pv, kc, vc, n), kw = of_case(1)
    a = fc.shared_prefix_attention(q, pk[:, :0], pv[:, :0], kc, vc, n, return_lse=True, **kw)
    b = fc.tree_attention(q, kc, vc, n, return_lse=True, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_slices_of_larger_buffers(gpu_device):
    """A prefix in a larger buffer, heads innermost, NaN behind it and behind the sequences' rows."""
    (q, pk, pv, kc, vc, n), kw = of_case(1)
    want = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
    buf = torch.full((900, 2, 2, 128), float("nan"), dtype=BF, device="cuda")
    buf[:700, 0], buf[:700, 1] = pk.transpose(0, 1), pv.transpose(0, 1)
    k2, v2 = buf[:700, 0].transpose(0, 1), buf[:700, 1].transpose(0, 1)
    kc, vc = kc.clone(), vc.clone()
    for b, x in enumerate(n.tolist()):
        kc[b, :, x + 8:], vc[b, :, x + 8:] = float("nan"), float("inf")
    got = fc.shared_prefix_attention(q, k2, v2, kc, vc, n, return_lse=True, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(2, 700, 129, dtype=BF, device="cuda")
    odd[..., 1:] = pk
    got = fc.shared_prefix_attention(q, odd[..., 1:], v2, kc, vc, n, return_lse=True, **kw)  # copied by the call
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("i", [1, 13, 18])
def test_lengths_that_do_not_fit(gpu_device, i):
    """NaN for the sequences whose rows do not fit, and for them alone; also under a window."""
    (q, pk, pv, kc, vc, n), kw = of_case(i)
    for window in (0, 100):
        kw = dict(kw, sliding_window=window)
        good = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
        m = n.clone()
        m[0], m[1] = kc.shape[2], -5
        o, lse = fc.shared_prefix_attention(q, pk, pv, kc, vc, m, return_lse=True, **kw)
        assert bool(torch.isnan(o[:2]).all()) and bool(torch.isnan(lse[:2]).all())
        assert torch.equal(torch.isnan(o[2:]), torch.isnan(good[0][2:]))
        # (lengths choose the chunks, and so the order of the sums: two roundings to the type apart at most)
        assert torch.allclose(o[2:].float(), good[0][2:].float(), rtol=2 * torch.finfo(o.dtype).eps,
                              atol=2 * torch.finfo(o.dtype).eps)
        assert torch.allclose(lse[2:], good[1][2:], rtol=2.0 ** -20, atol=2.0 ** -20)


def test_a_row_that_is_not_a_number(gpu_device):
    (q, pk, pv, kc, vc, n), kw = of_case(12)
    good = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, **kw)
    q2 = q.clone()
    q2[5, 3, 0, 7] = float("nan")
    o = fc.shared_prefix_attention(q2, pk, pv, kc, vc, n, **kw)
    assert bool(torch.isnan(o[5, 3]).all())
    o[5, 3] = good[5, 3]
    assert torch.equal(o, good)
    pk2 = pk.clone()
    pk2[1, 999] = float("nan")
    o = fc.shared_prefix_attention(q, pk2, pv, kc, vc, n, **kw)
    assert bool(torch.isnan(o[:, 4:]).all()) and torch.equal(o[:, :4], good[:, :4])


@pytest.mark.parametrize("i", [0, 18])
def test_streams_and_graphs(gpu_device, i):
    (q, pk, pv, kc, vc, n), kw = of_case(i)
    want = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
    for turn in range(4):
        n.copy_((n + 7 * turn) % (kc.shape[2] + 1))  # (also lengths that leave no room)
        pk.copy_(draw(turn, 1, *pk.shape, pk.dtype)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, return_lse=True, **kw)
        for x, y in zip(out, want):
            assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(), y.nan_to_num())


def test_empty_and_refused(gpu_device):
    (q, pk, pv, kc, vc, n), _ = of_case(0)
    o, lse = fc.shared_prefix_attention(q[:, :, :0], pk, pv, kc, vc, n, return_lse=True)
    assert o.shape == (2, 8, 0, 128) and lse.shape == (2, 8, 0)
    ok = dict(query=q, prefix_key=pk, prefix_value=pv, key_cache=kc, value_cache=vc, lengths=n)
    for kw in (dict(prefix_key=pk.half()), dict(prefix_value=pv.cpu()), dict(prefix_key=pk.clone().requires_grad_()),
               dict(lengths=n.long()), dict(soft_cap=float("inf")), dict(query=q.float()),
               dict(tree_mask=torch.ones(2, 2, device="cuda", dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            fc.shared_prefix_attention(**dict(ok, **kw))
    for kw in (dict(prefix_key=pk[:1]), dict(prefix_value=pv[:, :299]), dict(prefix_key=pk[None], prefix_value=pv[None]),
               dict(prefix_key=pk[:1], prefix_value=pv[:1]), dict(query=q[:, :7])):
        with pytest.raises(AssertionError):
            fc.shared_prefix_attention(**dict(ok, **kw))


MANY = [
    # dtype, B, Hq, Hkv, T, P, C, lengths, mask, window, cap, scale: eight row tiles of the prefix and more
    (BF, 64, 8, 1, 1, 1500, 40, [i % 40 for i in range(64)], None, 0, 0.0, None),
    (FH, 30, 8, 1, 8, 700, 30, [i % 22 for i in range(30)], "batch", 0, 0.0, None),     # two row tiles a sequence
    (BF, 32, 16, 2, 1, 63, 70, [2 * i for i in range(32)], None, 50, 0.0, None),       # windows that end in the prefix or behind
    (FH, 64, 4, 1, 1, 1, 9, [i % 9 for i in range(64)], None, 0, 30.0, 0.11),
    (BF, 63, 4, 1, 1, 2049, 40, [i % 44 - 2 for i in range(63)], None, 1000, 0.0, None),  # sequences that do not fit
    (FH, 43, 12, 2, 2, 640, 20, [i % 19 for i in range(43)], "shared", 333, 20.0, -0.2),
    (BF, 16, 16, 1, 1, 8200, 3, [i % 3 for i in range(16)], None, 0, 0.0, 0.0),
    (BF, 100, 10, 2, 3, 129, 300, [3 * i - 3 for i in range(100)], "holes", 70, 0.0, -0.09),
]


@pytest.mark.parametrize("i", range(len(MANY)))
def test_many_sequences(gpu_device, i):
    dtype, B, Hq, Hkv, T, P, C, n, mask, window, cap, scale = MANY[i]
    q, kc, vc = (draw(s + i, B, h, r, 128, dtype, "bsnd") for s, h, r in ((1, Hq, T), (50, Hkv, C), (90, Hkv, C)))
    big = torch.full((2, Hkv, P + 40, 128), float("nan"), dtype=dtype, device="cuda")  # a prefix shorter than its buffer
    big[0, :, 3:3 + P], big[1, :, 3:3 + P] = draw(130 + i, 1, Hkv, P, 128, dtype)[0], draw(170 + i, 1, Hkv, P, 128, dtype)[0]
    pk, pv = big[0, :, 3:3 + P], big[1, :, 3:3 + P]
    m = depths = None
    if mask:
        made = [tree(T, 7 * i + b, mask) for b in range(B if mask in ("batch", "holes") else 1)]
        m = torch.stack([x for x, _ in made])
        depths = torch.stack([d for _, d in made]).expand(B, T)
    lengths = torch.tensor(n, dtype=torch.int32)
    args = (q, pk, pv, kc, vc, lengths.cuda())
    kw = dict(tree_mask=None if m is None else m.cuda(), depths=None if m is None else depths.cuda(), sliding_window=window,
              soft_cap=cap, scale=scale)
    o, lse = fc.shared_prefix_attention(*args, return_lse=True, **kw)
    ro, rl, to, tl = oracle(q, pk, pv, kc, vc, lengths, m, depths, dict(sliding_window=window, scale=scale, soft_cap=cap), dtype)
    fits = (lengths >= 0) & (lengths + T <= C)
    check("o", o[fits.cuda()], ro[fits], to[fits])
    check("lse", lse[fits.cuda()], rl[fits], tl[fits])
    assert bool(o[~fits.cuda()].isnan().all()) and bool(lse[~fits.cuda()].isnan().all())
    again = fc.shared_prefix_attention(*args, return_lse=True, **kw)
    assert torch.equal(o[fits.cuda()], again[0][fits.cuda()]) and torch.equal(lse[fits.cuda()], again[1][fits.cuda()])
    if i == 0:
        q[5, 3] = float("nan")  # a row that is not a number leaves the others
        x = fc.shared_prefix_attention(*args, **kw)
        assert bool(x[5, 3].isnan().all())
        x[5, 3] = o[5, 3]
        assert torch.equal(x, o)


def test_many_sequences_in_a_graph(gpu_device):
    """Captured once and replayed as lengths and queries change, on another stream too: what an eager call gives."""
    B, T, P, C = 64, 1, 900, 50
    q, kc, vc = (draw(s, B, h, r, 128, FH, "bsnd") for s, h, r in ((1, 16, T), (50, 4, C), (90, 4, C)))
    pk, pv = draw(130, 1, 4, P, 128, FH)[0], draw(170, 1, 4, P, 128, FH)[0]
    n = torch.arange(B, dtype=torch.int32, device="cuda") % 40
    args = (q, pk, pv, kc, vc, n)
    want = fc.shared_prefix_attention(*args, sliding_window=700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fc.shared_prefix_attention(*args, sliding_window=700)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fc.shared_prefix_attention(*args, sliding_window=700, return_lse=True)
    for turn in range(3):
        q.copy_(draw(10 + turn, B, 16, T, 128, FH))
        n.copy_(torch.arange(B, dtype=torch.int32) * (7 + turn) % 49)
        graph.replay()
        torch.cuda.synchronize()
        want = fc.shared_prefix_attention(*args, sliding_window=700, return_lse=True)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
