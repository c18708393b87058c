"""Eviction on the GPU: which rows stay is compared with the host's sort, and the copies bit by bit."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # dtype, B, H, C, D, keep, recent, sinks, lengths, scores
    (BF, 2, 2, 300, 128, 100, 10, 4, [300, 80], "random"),
    (FH, 3, 1, 2000, 64, 500, 0, 0, [2000, 501, 500], "random"),
    (FS, 1, 3, 1500, 32, 700, 33, 1, [1499], "ties"),
    (BF, 1, 2, 5000, 256, 7, 3, 4, [5000], "random"),              # nothing goes by score
    (BF, 1, 1, 64, 128, 1, 0, 0, [64], "random"),
    (FH, 2, 2, 1030, 64, 1029, 0, 5, [1030, 0], "ties"),
    (FS, 1, 1, 4097, 256, 1000, 100, 0, [4097], "special"),
    (BF, 2, 1, 40, 32, 50, 20, 20, [40, 13], "random"),             # a budget beyond the cache
    (BF, 1, 1, 3000, 64, 1024, 0, 0, [3000], "equal"),
    (BF, 2, 2, 257, 64, 128, 1, 0, [1000000, -5], "special"),       # lengths outside the cache
    (FH, 2, 1, 20001, 32, 5000, 100, 4, [20001, 8200], "random"),    # several blocks of slots
    (BF, 1, 2, 9000, 32, 1500, 0, 3, [9000], "special"),
    (BF, 1, 1, 30000, 32, 12000, 64, 0, [29999], "ties"),
    (BF, 1, 1, 16500, 32, 100, 20, 70, [16500], "random"),
]


def scores_of(kind, B, H, C, seed):
    g = torch.Generator().manual_seed(seed)
    s = torch.exp(3 * torch.randn(B, H, C, generator=g))
    if kind == "ties":
        s = (s * 2).round().clamp(max=6) / 4
    elif kind == "equal":
        s = torch.full((B, H, C), 0.25)
    elif kind == "special":
        s = s - 5.0
        for i, x in enumerate((float("nan"), float("inf"), float("-inf"), 0.0, -0.0, 1e-42, -1e-42, -float("nan"))):
            s[..., 3 + i::17] = x
    return s


def draw(seed, B, H, S, D, dtype, layout="bnsd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "bsnd":
        return torch.randn(B, S, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    return torch.randn(B, H, S, D, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_the_host(gpu_device, i, given):
    dtype, B, H, C, D, keep, recent, sinks, lengths, kind = CASES[i]
    layout = "bsnd" if i % 2 else "bnsd"
    k, v = draw(i, B, H, C, D, dtype, layout), draw(20 + i, B, H, C, D, dtype, layout)
    s = scores_of(kind, B, H, C, 40 + i)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, rows = None, keep
    if given:  # a larger cache in another layout, its old rows stay behind
        rows = keep + 37
        out = (draw(60, B, H, rows, D, dtype, "bsnd"), draw(61, B, H, rows, D, dtype), torch.full((B, H, rows), 7.0).cuda())
    before = None if out is None else [x.cpu() for x in out]
    ko, vo, so, slots, m = fc.evict_cache(k, v, s.cuda(), n, keep, recent=recent, sinks=sinks, out=out)
    if given:
        assert ko is out[0] and vo is out[1] and so is out[2]
    assert ko.shape == (B, H, rows, D) and so.shape == (B, H, rows) and slots.shape == (B, H, keep)
    kc, vc = k.cpu(), v.cpu()
    bits = lambda x: x.cpu().contiguous().view(torch.int32)  # noqa: E731
    for b in range(B):
        live = min(max(lengths[b], 0), C)
        for h in range(H):
            want = orc.evict(s[b, h].tolist(), live, keep, recent, sinks)
            x = len(want)
            assert int(m[b]) == x and slots[b, h, :x].tolist() == want and slots[b, h, x:].tolist() == [-1] * (keep - x)
            assert torch.equal(ko[b, h, :x].cpu(), kc[b, h, want]) and torch.equal(vo[b, h, :x].cpu(), vc[b, h, want])
            assert torch.equal(bits(so[b, h, :x]), bits(s[b, h, want])) and float(so[b, h, x:].abs().sum()) == 0.0
            if given:
                assert torch.equal(ko[b, h, x:].cpu(), before[0][b, h, x:])
                assert torch.equal(vo[b, h, x:].cpu(), before[1][b, h, x:])
            else:
                assert float(ko[b, h, x:].float().abs().sum()) == float(vo[b, h, x:].float().abs().sum()) == 0.0


def test_long_caches(gpu_device):
    """Every digit of the search counts: scores that differ in their last bits only, and heavy ties."""
    C = 70001
    k = draw(1, 1, 2, C, 32, BF)
    near = (torch.randperm(C, generator=torch.Generator().manual_seed(1)).int() + 0x3f800000).view(torch.float32)
    many = (torch.arange(C) * 7919 % 5).float()
    s = torch.stack((near, many))[None]
    n = torch.tensor([C], dtype=torch.int32, device="cuda")
    for keep in (1, 1000, 40000, C - 1):
        ko, _, _, slots, _ = fc.evict_cache(k, k, s.cuda(), n, keep)
        for h in range(2):
            want = orc.evict(s[0, h].tolist(), C, keep, 0, 0)
            assert slots[0, h].tolist() == want and torch.equal(ko[0, h].cpu(), k[0, h].cpu()[want])


def test_refusals(gpu_device):
    k, s = draw(1, 1, 2, 50, 64, BF), torch.rand(1, 2, 50).cuda()
    n = torch.tensor([50], dtype=torch.int32, device="cuda")
    new = lambda rows=20, D=64: (torch.zeros(1, 2, rows, D, dtype=BF, device="cuda"),  # noqa: E731
                                 torch.zeros(1, 2, rows, D, dtype=BF, device="cuda"), torch.zeros(1, 2, rows, device="cuda"))
    bad = [dict(keep=0), dict(keep=10, recent=6, sinks=5), dict(keep=10, recent=-1), dict(keep=10, scores=s.half()),
           dict(keep=10, scores=s[..., :49]), dict(keep=10, scores=s.cpu()), dict(keep=10, lengths=n.long()),
           dict(keep=30, out=new()), dict(keep=10, out=new(D=32)), dict(keep=10, out=new()[:2] + (s,)),
           dict(keep=10, out=(k, k.clone(), s.clone())),                       # the old cache itself
           dict(keep=10, out=(k[:, :, 30:], new()[1], new()[2])),              # and a part of it
           dict(keep=10, out=(new()[0][:, :1].expand(1, 2, 20, 64),) + new()[1:]),
           dict(keep=10, key_cache=k.clone().requires_grad_())]
    for kw in bad:
        args = dict(key_cache=k, value_cache=k, scores=s, lengths=n)
        args.update(kw)
        with pytest.raises((RuntimeError, ValueError)):
            fc.evict_cache(**args)
    with pytest.raises(AssertionError):
        fc.evict_cache(k, k[:, :1], s, n, 10)
    with pytest.raises(RuntimeError):
        fc.evict_cache(k[:, :, :0], k[:, :, :0], s[..., :0], n, 10)


def test_graph_replays(gpu_device):
    k, v = draw(1, 2, 2, 900, 64, BF), draw(2, 2, 2, 900, 64, BF)
    s, n = torch.rand(2, 2, 900).cuda(), torch.tensor([900, 100], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fc.evict_cache(k, v, s, n, 300, recent=10)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = fc.evict_cache(k, v, s, n, 300, recent=10)
    for rep, (a, b) in enumerate(((900, 100), (301, 300), (20, 899))):
        n.copy_(torch.tensor([a, b], dtype=torch.int32))
        s.copy_(torch.rand(2, 2, 900, generator=torch.Generator().manual_seed(rep)))
        eager = fc.evict_cache(k, v, s, n, 300, recent=10)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, eager):
            assert torch.equal(x, y)
