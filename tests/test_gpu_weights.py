"""Attention weight sums on the GPU against the float64 oracle (tolerances: oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
import npu_flash_attention as nfa
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # dtype, B, Hq, Hkv, Sq, Skv, D, causal, start, lengths, window, cap
    (BF, 2, 8, 2, 1, 500, 128, False, 0, [500, 33], 0, 0.0),
    (BF, 1, 8, 2, 300, 300, 128, True, 0, None, 0, 0.0),
    (FH, 2, 7, 1, 32, 1000, 64, True, 968, None, 0, 30.0),
    (FH, 1, 4, 4, 129, 129, 64, True, 0, None, 20, 0.0),
    (BF, 2, 4, 2, 40, 260, 256, False, 0, [0, 200], 0, 50.0),
    (BF, 2, 3, 1, 65, 65, 32, True, 0, [65, 30], 0, 0.0),
    (FS, 1, 4, 2, 70, 200, 128, True, 130, None, 50, 0.0),
    (FS, 2, 2, 2, 1, 90, 64, False, 0, [90, 1], 0, 30.0),
    (FS, 1, 2, 1, 33, 40, 256, True, 7, None, 0, 0.0),
    (FS, 1, 3, 3, 5, 31, 32, True, 0, None, 0, 0.0),
    (BF, 2, 4, 1, 10, 100, 64, True, [90, -4], [100, 95], 30, 0.0),   # own starts; rows that see nothing
    (FH, 1, 2, 1, 700, 600, 128, True, 0, None, 100, 0.0),            # rows behind every key's window
    (BF, 1, 16, 1, 3, 5000, 128, True, 4997, None, 0, 0.0),
    (BF, 1, 1, 1, 1, 1, 32, True, 0, None, 0, 0.0),
    (FH, 1, 5, 1, 900, 70, 64, False, 0, None, 0, 0.0),               # few keys, many rows, five heads a key
    (BF, 2, 11, 1, 401, 300, 128, True, [0, -390], [300, 7], 0, 20.0),
    (FS, 1, 6, 2, 500, 40, 256, False, 0, [33], 0, 0.0),
]


def draw(seed, B, H, S, D, dtype, layout="bnsd"):
    g = torch.Generator().manual_seed(seed)
    if layout == "bsnd":
        return torch.randn(B, S, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    return torch.randn(B, H, S, D, generator=g).to(dtype).cuda()


def lse_of(q, k, causal, starts, lengths, window, scale, cap):
    """The rows' LSE in float64, -inf for rows without keys."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.empty(B, Hq, Sq, dtype=torch.float64)
    for b in range(B):
        n = k.shape[2] if lengths is None else lengths[b]
        s0 = starts[b] if isinstance(starts, list) else starts
        i, j = torch.arange(Sq)[:, None] + s0, torch.arange(n)[None]
        hide = torch.zeros(Sq, n, dtype=torch.bool)
        if causal:
            hide |= j > i
        if window:
            hide |= i - j > window
        for h in range(Hq):
            x = q[b, h].double() @ k[b, h // G, :n].double().T * scale
            x = cap * torch.tanh(x / cap) if cap else x
            out[b, h] = torch.logsumexp(x.masked_fill(hide, float("-inf")), dim=-1)
    return out


def check(x, ref, tol):
    x = x.cpu().double()
    worst = ((x - ref).abs() / tol).max().item()
    assert bool(torch.isfinite(x).all()) and worst <= 1.0, f"{worst:.2f} tolerances"


@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_oracle(gpu_device, i):
    dtype, B, Hq, Hkv, Sq, Sk, D, causal, start, lengths, window, cap = CASES[i]
    layout = "bsnd" if i % 2 else "bnsd"
    q, k = draw(i, B, Hq, Sq, D, dtype, layout), draw(30 + i, B, Hkv, Sk, D, dtype, layout)
    scale = 0.13
    lse = lse_of(q.cpu(), k.cpu(), causal, start, lengths, window, scale, cap).float()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s0 = torch.tensor(start, dtype=torch.int32, device="cuda") if isinstance(start, list) else start
    kw = dict(causal=causal, query_start=s0, lengths=n, sliding_window=window, scale=scale, soft_cap=cap)
    w = fc.attention_weight_sums(q, k, lse.cuda(), **kw)
    starts = torch.tensor(start) if isinstance(start, list) else start
    ref, tol = orc.weight_sums(q.cpu(), k.cpu(), lse, causal, starts, lengths, window, scale, cap)
    check(w, ref, tol)
    assert torch.equal(w, fc.attention_weight_sums(q, k, lse.cuda(), **kw))
    # added to what is there; keys left out keep what they had
    base = torch.rand(B, Hkv, Sk, generator=torch.Generator().manual_seed(4)).cuda()
    into = base.clone()
    assert fc.attention_weight_sums(q, k, lse.cuda(), into=into, **kw) is into
    check(into, ref + base.cpu().double(), tol + (ref + base.cpu().double()) * 2.0 ** -23)
    if lengths is not None:
        for b, x in enumerate(lengths):
            assert torch.equal(into[b, :, x:], base[b, :, x:]) and float(w[b, :, x:].abs().sum()) == 0.0


def test_with_the_forward_lse_every_row_gives_one(gpu_device):
    """With the forward's own LSE the weights of a row add up to 1, so all sums to G * Sq per KV head: the sums' and
    LSE's tolerances beside bf16 inputs, under 2^-12 of it."""
    q, k = draw(1, 2, 8, 333, 128, BF), draw(2, 2, 2, 333, 128, BF)
    _, lse = nfa.npu_flash_attention_forward(q, k, k, causal=True, return_lse=True)
    w = fc.attention_weight_sums(q, k, lse, causal=True)
    total = w.double().sum(-1)
    assert bool(((total - 4 * 333).abs() <= 4 * 333 * 2.0 ** -12).all())


def test_rows_without_keys_and_nan(gpu_device):
    q, k = draw(1, 1, 2, 40, 64, BF), draw(2, 1, 1, 64, 64, BF)
    lse = torch.zeros(1, 2, 40, device="cuda")
    lse[:, :, ::2] = float("-inf")
    w = fc.attention_weight_sums(q, k, lse, causal=True, query_start=24)
    ref, tol = orc.weight_sums(q.cpu(), k.cpu(), lse.cpu(), True, 24)
    check(w, ref, tol)
    none = fc.attention_weight_sums(q, k, torch.full_like(lse, float("-inf")))
    assert float(none.abs().sum()) == 0.0
    k[0, 0, 50] = float("nan")  # behind the length: nothing
    n = torch.tensor([50], dtype=torch.int32, device="cuda")
    x = fc.attention_weight_sums(q, k, lse, causal=True, query_start=24, lengths=n)
    assert torch.equal(x[..., :50], w[..., :50]) and float(x[..., 50:].abs().sum()) == 0.0
    y = fc.attention_weight_sums(q, k, lse, causal=True, query_start=24)  # that key's sum alone
    assert bool(torch.isnan(y[0, 0, 50])) and torch.equal(y[..., :50], w[..., :50]) and torch.equal(y[..., 51:], w[..., 51:])
    for out_of_range, like in ((1000, 64), (-7, 0)):
        n.fill_(out_of_range)
        a = fc.attention_weight_sums(q, k.nan_to_num(), lse, lengths=n)
        b = fc.attention_weight_sums(q, k.nan_to_num(), lse, lengths=torch.full_like(n, like))
        assert torch.equal(a, b)


def test_refusals(gpu_device):
    q, k = draw(1, 2, 4, 3, 64, BF), draw(2, 2, 2, 20, 64, BF)
    lse, n = torch.zeros(2, 4, 3, device="cuda"), torch.tensor([4, 5], dtype=torch.int32, device="cuda")
    for kw in (dict(lengths=n.long()), dict(query_start=n.cpu()), dict(query_start=1 << 40),
               dict(into=torch.zeros(2, 2, 19, device="cuda")), dict(into=torch.zeros(2, 2, 20)),
               dict(into=torch.zeros(2, 2, 40, device="cuda")[..., ::2]), dict(scale=float("inf"))):
        with pytest.raises(RuntimeError):
            fc.attention_weight_sums(q, k, lse, **kw)
    with pytest.raises(RuntimeError, match="gradient"):
        fc.attention_weight_sums(q.clone().requires_grad_(), k, lse)
    with pytest.raises(RuntimeError):
        fc.attention_weight_sums(q, k, lse.cpu())
    with pytest.raises(AssertionError):
        fc.attention_weight_sums(q, k, lse[..., :2])
    assert float(fc.attention_weight_sums(q[:, :, :0], k, lse[:, :, :0]).sum()) == 0.0
    assert fc.attention_weight_sums(q, k[:, :, :0], lse).shape == (2, 2, 0)


def test_graph_replays(gpu_device):
    q, k = draw(1, 2, 8, 4, 128, BF), draw(2, 2, 2, 700, 128, BF)
    lse, n = torch.full((2, 8, 4), 3.0, device="cuda"), torch.tensor([700, 9], dtype=torch.int32, device="cuda")
    start = torch.tensor([696, 5], dtype=torch.int32, device="cuda")
    into = torch.zeros(2, 2, 700, device="cuda")
    call = lambda x: fc.attention_weight_sums(q, k, lse, causal=True, query_start=start, lengths=n, into=x)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(into.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(into)
    into.zero_()
    eager = torch.zeros_like(into)
    for a, b in ((700, 9), (300, 640), (20, 700)):
        n.copy_(torch.tensor([a, b], dtype=torch.int32))
        start.copy_(n - 4)
        call(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(into, eager)


@pytest.mark.parametrize("dtype", [BF, FH, FS])
@pytest.mark.parametrize("top", [8.0, 40.0])
def test_soft_cap_to_the_last_bits(gpu_device, dtype, top):
    """One query row and keys along one element, so that the scores s are exact, and LSE 0: weights exp(cap tanh(s / cap)).
    The capped score is off by 9 half steps of itself (scale / cap, the quotient, the series, cap log2 e) up to |s| = cap / 4,
    and by another 4 of the cap above (1 - 2 / (1 + e^2y): exponential, sum, reciprocal, difference); exp2 by a step."""
    s = torch.linspace(-top, top, 301).to(dtype)
    q, k = torch.zeros(1, 1, 1, 64, dtype=dtype), torch.zeros(1, 1, 301, 64, dtype=dtype)
    q[..., 0], k[0, 0, :, 0] = 1.0, s
    w = fc.attention_weight_sums(q.cuda(), k.cuda(), torch.zeros(1, 1, 1, device="cuda"), scale=1.0, soft_cap=30.0)
    x = 30.0 * torch.tanh(s.double() / 30.0)
    h = 2.0 ** -24
    tol = 9 * h * x.abs() + torch.where(s.double().abs() > 7.4, 4 * h * 30.0, 0.0) + 2 * h
    worst = ((w[0, 0].cpu().double() / torch.exp(x) - 1.0).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.2f} tolerances"
