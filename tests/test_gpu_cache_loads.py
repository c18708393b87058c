"""What the rotary, weight-sum and eviction kernels do only where there are many tokens, heads or keys: several heads per
thread, two blocks of keys per workgroup, several rounds of copies.  Which sizes reach it is each launcher's own rule,
restated here for the card's number of CUs, so that a case that no longer reaches it fails.  The oracle runs in float64 on
the GPU."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def draw(seed, B, H, S, D, dtype, layout="bnsd"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "bsnd":
        return torch.randn(B, S, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    return torch.randn(B, H, S, D, generator=g, device="cuda").to(dtype)


def check(x, ref, tol, what=""):
    x = x.detach().double()
    worst = ((x - ref).abs() / tol).max().item()
    assert bool(torch.isfinite(x).all()) and worst <= 1.0, f"{what}: {worst:.2f} tolerances"


# ------------------------------------------------------------------------------------------------------- rotation --
def heads_per_thread(tokens, heads, D, dtype, pairs):
    chunk = 16 // dtype.itemsize
    if pairs % chunk == 0:
        per_block = 256 // (D // (2 * chunk))
        blocks = -(-tokens // per_block)
    else:
        blocks = -(-tokens * (D // 2) // 256)
    hpt = -(-heads // min(-(-1024 // blocks), heads))
    return hpt if hpt <= 2 else -(-hpt // 4) * 4


ROTARY = [
    # dtype, B, Hq, Hkv, S, D, pairs, interleaved, layout, heads per thread
    (BF, 1, 37, 3, 2570, 64, 32, False, "bnsd", 2),      # rounds of two
    (BF, 1, 37, 3, 4500, 64, 32, True, "bnsd", 4),       # one whole round
    (FH, 1, 11, 2, 16500, 64, 16, False, "bsnd", 4),     # the last thread has one head
    (FH, 2, 10, 3, 5000, 256, 128, False, "bnsd", 8),    # two rounds; the second thread's last one has one head
    (BF, 1, 40, 10, 4200, 256, 128, True, "bnsd", 16),   # four rounds; the last thread has two heads
    (FS, 1, 4, 1, 33000, 64, 32, False, "bnsd", 8),      # one thread has all heads, and a part of a round
    (FS, 2, 5, 2, 16500, 32, 8, True, "bsnd", 4),
    (BF, 1, 11, 2, 4480, 64, 5, False, "bnsd", 8),       # the general kernel
    (FS, 2, 7, 4, 5000, 64, 31, True, "bsnd", 12),
]


@pytest.mark.parametrize("i", range(len(ROTARY)))
def test_rotary_with_several_heads_per_thread(gpu_device, i):
    dtype, B, Hq, Hkv, S, D, pairs, inter, layout, hpt = ROTARY[i]
    assert heads_per_thread(B * S, Hq + Hkv, D, dtype, pairs) == hpt
    q, k = draw(i, B, Hq, S, D, dtype, layout).requires_grad_(), draw(50 + i, B, Hkv, S, D, dtype, layout).requires_grad_()
    gq, gk = draw(100 + i, B, Hq, S, D, dtype), draw(150 + i, B, Hkv, S, D, dtype, layout)
    f, m = rot.rotary_frequencies(2 * pairs, scaling="yarn", factor=4.0, original_length=512, device="cuda")
    pos = torch.randint(0, 100000, (B, S), generator=torch.Generator().manual_seed(i)).cuda()
    yq, yk = rot.rotary_embedding(q, k, f, positions=pos, interleaved=inter, magnitude=m)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for what, x, y, inv in (("q", q, yq, False), ("k", k, yk, False), ("dq", gq, dq, True), ("dk", gk, dk, True)):
        ref, slack = orc.rotary(x.detach().double(), f, pos, inter, m, inv)
        check(y, ref, orc.rounded(ref, slack, dtype), what)
        assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])


APPENDS = [
    # dtype, B, Hq, Hkv, S, C, D, pairs, lengths, heads per thread (rounds mix query, key and value heads)
    (FH, 2, 9, 3, 8250, 9000, 64, 32, [0, 750], 4),
    (BF, 3, 9, 3, 6000, 6500, 128, 32, [500, 100, 499], 8),
    (BF, 1, 7, 1, 2600, 2600, 64, 32, [0], 1),
    (FS, 2, 6, 3, 3000, 4000, 64, 32, [1000, 900], 2),
    (FS, 1, 4, 2, 9000, 9001, 32, 15, [1], 4),           # the general kernel
]


@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append_with_several_heads_per_thread(gpu_device, i):
    dtype, B, Hq, Hkv, S, C, D, pairs, n, hpt = APPENDS[i]
    assert heads_per_thread(B * S, Hq + 2 * Hkv, D, dtype, pairs) == hpt
    q, k, v = (draw(10 * i + j, B, h, S, D, dtype, "bsnd") for j, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    kc, vc = draw(10 * i + 4, B, Hkv, C, D, dtype), draw(10 * i + 5, B, Hkv, C, D, dtype)
    k0, v0 = kc.clone(), vc.clone()
    f, m = rot.rotary_frequencies(2 * pairs, device="cuda")
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    out = fc.rotary_append(q, k, v, kc, vc, lengths, f, interleaved=bool(i % 2), magnitude=1.125)
    pos = lengths.long()[:, None] + torch.arange(S, device="cuda")
    ref, slack = orc.rotary(q.double(), f, pos, bool(i % 2), 1.125)
    check(out, ref, orc.rounded(ref, slack, dtype), "q")
    ref, slack = orc.rotary(k.double(), f, pos, bool(i % 2), 1.125)
    tol = orc.rounded(ref, slack, dtype)
    for b, x in enumerate(n):
        check(kc[b, :, x:x + S], ref[b], tol[b], "key")
        assert torch.equal(vc[b, :, x:x + S], v[b])
        for new, old in ((kc, k0), (vc, v0)):
            assert torch.equal(new[b, :, :x], old[b, :, :x]) and torch.equal(new[b, :, x + S:], old[b, :, x + S:])


# ---------------------------------------------------------------------------------------------------- weight sums --
def weight_plan(dtype, B, Hq, Hkv, Sq, Sk, D, causal, start, window):
    """(1 where a workgroup has two blocks of keys, the parts of their query rows, the number of blocks)."""
    cus, row = torch.cuda.get_device_properties(0).multi_processor_count, D * dtype.itemsize
    keys = 256 if row <= 512 else 128
    blocks, bh, slots = -(-Sk // keys), B * Hkv, (1 if row >= 512 else 2) * cus
    start = Sk - Sq if isinstance(start, list) else start

    def tiles(x):
        lo, hi = max(x * keys - start if causal else 0, 0), Sq
        hi = min(hi, (x + 1) * keys + window - start) if window else hi
        return -(-(hi - lo) * (Hq // Hkv) // 32) if hi > lo else 0

    ends = [(tiles(x), tiles(blocks - 1 - x) if blocks - 1 - x != x else 0) for x in (0, blocks // 4, (blocks - 1) // 2)]
    one, two = max(max(e) for e in ends), max(sum(e) for e in ends)
    best = None
    for pair in (1, 0) if blocks > 1 else (0,):
        groups, work = ((blocks + 1) // 2 if pair else blocks) * bh, two if pair else one
        for n in range(1, 65):
            if n > 1 and one // n < (2 if dtype.itemsize == 2 else 1):
                break
            cost = -(-groups * n // slots) * (-(-work // n) + (9 if pair else 5))
            if best is None or cost < best[0]:
                best = cost, pair, n
    return best[1], best[2], blocks


WEIGHTS = [
    # dtype, B, Hq, Hkv, Sq, Skv, D, causal, start, lengths, window, cap
    (BF, 4, 32, 32, 40, 1250, 32, False, 0, [1250, 700, 513, 20], 0, 0.0),   # an odd number of blocks: the middle one alone
    (BF, 4, 32, 32, 1, 1025, 128, False, 0, [1025, 1024, 0, 257], 0, 30.0),  # one key in the last block
    (FH, 8, 16, 16, 70, 1500, 32, True, 1430, None, 0, 0.0),                 # an even number
    (FH, 8, 16, 16, 70, 1300, 32, True, 1230, [1300, 1281, 1280, 1279, 1025, 1024, 1, 400], 300, 0.0),
    (BF, 2, 32, 8, 1500, 1500, 32, True, 0, None, 0, 0.0),                   # pairs in parts
    (FH, 1, 16, 4, 2000, 2100, 64, True, 100, [1999], 0, 20.0),
    (BF, 2, 40, 8, 1100, 1700, 128, True, [600, -300], [1700, 1500], 0, 0.0),  # five heads a key, own starts
    (BF, 2, 28, 4, 1500, 3000, 64, True, 1500, None, 700, 0.0),
    (FS, 3, 32, 32, 2, 700, 128, True, 698, None, 0, 0.0),
    (FS, 2, 32, 32, 1, 1000, 256, False, 0, [1000, 897], 0, 0.0),            # rows of 1 KB: blocks of 128 keys
    (FS, 1, 24, 8, 900, 1500, 64, True, 200, None, 0, 30.0),
    (BF, 4, 32, 32, 3, 1000, 256, True, 997, None, 0, 50.0),
]


def lse_of(q, k, causal, starts, lengths, window, scale, cap):
    """The rows' LSE in float64, -inf for rows without keys."""
    B, Hq, Sq, D = q.shape
    out = torch.empty(B, Hq, Sq, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = k.shape[2] if lengths is None else lengths[b]
        i = torch.arange(Sq, device="cuda")[:, None] + (starts[b] if isinstance(starts, list) else starts)
        j = torch.arange(n, device="cuda")[None]
        hide = torch.zeros(Sq, n, dtype=torch.bool, device="cuda")
        if causal:
            hide |= j > i
        if window:
            hide |= i - j > window
        for h in range(Hq):
            x = q[b, h].double() @ k[b, h // (Hq // k.shape[1]), :n].double().T * scale
            x = cap * torch.tanh(x / cap) if cap else x
            out[b, h] = torch.logsumexp(x.masked_fill(hide, float("-inf")), dim=-1)
    return out


@pytest.mark.parametrize("i", range(len(WEIGHTS)))
def test_weight_sums_with_two_blocks_per_workgroup(gpu_device, i):
    dtype, B, Hq, Hkv, Sq, Sk, D, causal, start, lengths, window, cap = WEIGHTS[i]
    pair, parts, blocks = weight_plan(dtype, B, Hq, Hkv, Sq, Sk, D, causal, start, window)
    assert pair == 1
    print(f"{blocks} blocks of keys, parts {parts}")
    q, k = draw(i, B, Hq, Sq, D, dtype, "bsnd" if i % 2 else "bnsd"), draw(50 + i, B, Hkv, Sk, D, dtype)
    lse = lse_of(q, k, causal, start, lengths, window, 0.13, cap).float()
    lse[0, 0, Sq // 2] = float("-inf")  # a row that is taken as one without keys
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s0 = torch.tensor(start, dtype=torch.int32, device="cuda") if isinstance(start, list) else start
    kw = dict(causal=causal, query_start=s0, lengths=n, sliding_window=window, scale=0.13, soft_cap=cap)
    w = fc.attention_weight_sums(q, k, lse, **kw)
    with torch.device("cuda"):
        ref, tol = orc.weight_sums(q, k, lse, causal, torch.tensor(start) if isinstance(start, list) else start, lengths,
                                   window, 0.13, cap)
    check(w, ref, tol)
    assert torch.equal(w, fc.attention_weight_sums(q, k, lse, **kw))
    base = torch.rand(B, Hkv, Sk, generator=torch.Generator().manual_seed(4)).cuda()
    into = base.clone()
    assert fc.attention_weight_sums(q, k, lse, into=into, **kw) is into
    check(into, ref + base.double(), tol + (ref + base.double()) * 2.0 ** -23)
    for b, x in enumerate(lengths or []):
        assert torch.equal(into[b, :, x:], base[b, :, x:]) and float(w[b, :, x:].abs().sum()) == 0.0


# ------------------------------------------------------------------------------------------------------- eviction --
EVICT = [
    # dtype, B, H, C, D, keep, recent, sinks, lengths
    (BF, 8, 8, 2000, 128, 1001, 30, 4, [2000, 1999, 1001, 1000, 1700, 1, 1500, 1800]),  # 256 threads, eight slots each
    (FS, 16, 16, 700, 64, 555, 0, 0, [700 - 9 * b for b in range(16)]),
    (BF, 8, 8, 6000, 32, 5003, 100, 0, [6000, 5004, 5003, 100, 0, 5500, 5999, 5800]),   # 1024 threads
    (FH, 4, 16, 9000, 64, 3001, 64, 4, [9000, 8193, 3002, 7000]),                       # sixteen slots each
    (BF, 8, 8, 16600, 32, 4502, 10, 1, [16600, 16385, 4503, 4502, 9000, 12000, 16384, 30]),  # scores read again
]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("i", range(len(EVICT)))
def test_eviction_with_several_rounds_of_copies(gpu_device, i, given):
    dtype, B, H, C, D, keep, recent, sinks, lengths = EVICT[i]
    cus, threads = torch.cuda.get_device_properties(0).multi_processor_count, 256 if C <= 2048 else 1024
    rows = 4 * (threads // (D * dtype.itemsize // 16))  # that a workgroup copies in one round
    parts = max(1, min(-(-keep // rows), cus * (1 if threads == 1024 else 2) // (B * H)))
    assert keep // parts > rows and keep % parts and keep // parts % rows  # rounds, unequal shares, a part of a round
    k, v = draw(i, B, H, C, D, dtype, "bsnd"), draw(20 + i, B, H, C, D, dtype)
    s = torch.exp(2 * torch.randn(B, H, C, generator=torch.Generator().manual_seed(i)))
    s[:, ::2] = (s[:, ::2] * 2).round().clamp(max=9) / 4  # every other head with many equal ones
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, last = None, keep
    if given:
        last = keep + 5
        out = (draw(60, B, H, last, D, dtype, "bsnd"), draw(61, B, H, last, D, dtype), torch.full((B, H, last), 7.0).cuda())
    before = None if out is None else [x.clone() for x in out]
    ko, vo, so, slots, m = fc.evict_cache(k, v, s.cuda(), n, keep, recent=recent, sinks=sinks, out=out)
    for b in range(B):
        for h in range(H):
            want = torch.tensor(orc.evict(s[b, h].tolist(), lengths[b], keep, recent, sinks), dtype=torch.int32).cuda()
            x = len(want)
            assert int(m[b]) == x and torch.equal(slots[b, h, :x], want) and bool((slots[b, h, x:] == -1).all())
            at = want.long()
            assert torch.equal(ko[b, h, :x], k[b, h, at]) and torch.equal(vo[b, h, :x], v[b, h, at])
            assert torch.equal(so[b, h, :x].cpu(), s[b, h, at.cpu()]) and float(so[b, h, x:].abs().sum()) == 0.0
            for y, old in ((ko, 0), (vo, 1)):
                rest = before[old][b, h, x:] if given else torch.zeros_like(y[b, h, x:])
                assert torch.equal(y[b, h, x:], rest)
