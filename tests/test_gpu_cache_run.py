"""The cache operators one after the other, as a server uses them: a prompt is rotated and attended, the weight of its
keys summed, the cache cut to a budget, drafted tokens appended and attended as a tree, and the accepted ones kept.
Each step is held against the float64 oracle on the GPU's own inputs of that step."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
import npu_flash_attention as nfa
from gpu_helpers import TOL, err
from oracle import attention_oracle as aorc
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def near(x, ref, tol, what):
    worst = ((x.cpu().double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} tolerances"


@pytest.mark.parametrize("dtype,D,inter", [(torch.bfloat16, 128, False), (torch.float16, 64, True),
                                           (torch.float32, 128, False)])
def test_prompt_evict_draft_accept(gpu_device, dtype, D, inter):
    B, Hq, Hkv, S, keep, room, T = 2, 8, 2, 210, 96, 160, 7
    g = torch.Generator().manual_seed(11)
    new = lambda h, s: torch.randn(B, s, h, D, generator=g).to(dtype).cuda().transpose(1, 2)  # noqa: E731
    q, k, v = new(Hq, S), new(Hkv, S), new(Hkv, S)
    f, m = rot.rotary_frequencies(D // 2, scaling="turns", factor=4.0, original_length=64, fast=4.0, device="cuda")

    # the prompt
    q, k = rot.rotary_embedding(q, k, f, interleaved=inter, magnitude=m)
    o, lse = nfa.npu_flash_attention_forward(q, k, v, causal=True, return_lse=True)
    ro, rl = aorc.forward(q.cpu(), k.cpu(), v.cpu(), True)
    assert err(o, ro) <= TOL[dtype]["o"] and err(lse, rl) <= TOL[dtype]["lse"]
    w = fc.attention_weight_sums(q, k, lse, causal=True)
    rw, tw = orc.weight_sums(q.cpu(), k.cpu(), lse.cpu(), causal=True)
    near(w, rw, tw, "weights")

    # cut to the budget, into a cache with room to grow
    cache = (torch.empty(B, Hkv, room, D, dtype=dtype, device="cuda"), torch.empty(B, Hkv, room, D, dtype=dtype, device="cuda"),
             torch.empty(B, Hkv, room, device="cuda"))
    n = torch.tensor([S, 50], dtype=torch.int32, device="cuda")  # the second prompt was a short one, padded
    kc, vc, score, slots, n = fc.evict_cache(k, v, w, n, keep, recent=16, sinks=2, out=cache)
    assert n.tolist() == [keep, 50]
    for h in range(Hkv):
        want = orc.evict(w[0, h].tolist(), S, keep, 16, 2)
        assert slots[0, h].tolist() == want and torch.equal(kc[0, h, :keep], k[0, h, want])

    # drafted tokens: a tree whose tokens sit at the prompt's end plus their depth
    parents = [-1, 0, 0, 1, 1, 2, -1]
    mask, depth = torch.zeros(T, T, dtype=torch.bool), torch.zeros(T, dtype=torch.int32)
    for t, p in enumerate(parents):
        if p >= 0:
            mask[t], depth[t] = mask[p], depth[p] + 1
        mask[t, t] = True
    prompt = torch.tensor([S, 50], dtype=torch.int32, device="cuda")
    dq, dk, dv = new(Hq, T), new(Hkv, T), new(Hkv, T)
    pos = prompt[:, None] + depth.cuda()
    dq = fc.rotary_append(dq, dk, dv, kc, vc, n, f, positions=pos, interleaved=inter, magnitude=m)
    o, lse = fc.tree_attention(dq, kc, vc, n, mask.cuda(), return_lse=True)
    ro, rl, to, tl = orc.tree_attention(dq.cpu(), kc.cpu(), vc.cpu(), n.cpu(), mask, dtype=dtype)
    near(o, ro, to, "tree o")
    near(lse, rl, tl, "tree lse")

    # tokens 0, 1, 4 are accepted: their rows move behind the cached ones, their weight is added
    path = torch.tensor([0, 1, 4], device="cuda")
    rows = n[:, None].long() + path
    at = torch.arange(B, device="cuda")[:, None]
    first = n[:, None].long() + torch.arange(3, device="cuda")
    kc[at, :, first], vc[at, :, first] = kc[at, :, rows], vc[at, :, rows]
    before = score.clone()
    fc.attention_weight_sums(dq[:, :, path], kc, lse[:, :, path].contiguous(), causal=True, query_start=n, lengths=n + 3,
                             into=score)
    rw, tw = orc.weight_sums(dq[:, :, path].cpu(), kc.cpu(), lse[:, :, path].cpu(), True, n.cpu(), (n + 3).cpu())
    near(score, before.cpu().double() + rw, tw + score.cpu().double() * 2.0 ** -23, "weights of the accepted")
    # each accepted row attended the cached keys and its own path: their weights add up to one
    total = (score - before).double().sum(-1).cpu()
    assert bool(((total - 3 * Hq // Hkv).abs() <= 3 * Hq // Hkv * 2.0 ** -10).all())
    n += 3
    kc2, vc2, score2, slots, n2 = fc.evict_cache(kc, vc, score, n, keep, recent=16)
    assert n2.tolist() == [keep, 53] and slots[1, 0, :53].tolist() == list(range(53))
    assert bool((slots[0, :, -16:] == torch.arange(keep + 3 - 16, keep + 3, device="cuda")).all())


def test_offsets_past_32_bits(gpu_device):
    """Caches whose rows lie 2^22 elements apart, so that row 520 starts past 2^31: as from dense ones, bit for bit."""
    D, C = 64, 600
    g = torch.Generator().manual_seed(3)
    new = lambda *s: torch.randn(*s, D, generator=g).bfloat16().cuda()  # noqa: E731
    wide = torch.zeros(C << 22, dtype=torch.bfloat16, device="cuda").view(1, 1, C, 1 << 22)
    far = [wide[..., 64 * i:64 * i + 64] for i in range(4)]
    k, v = new(1, 1, C), new(1, 1, C)
    far[0].copy_(k), far[1].copy_(v)
    n = torch.tensor([590], dtype=torch.int32, device="cuda")
    f, _ = rot.rotary_frequencies(D, device="cuda")
    q, k1, v1 = new(1, 2, 5), new(1, 1, 5), new(1, 1, 5)
    a = fc.rotary_append(q, k1, v1, k, v, n, f)
    b = fc.rotary_append(q, k1, v1, far[0], far[1], n, f)
    assert torch.equal(a, b) and torch.equal(far[0], k) and torch.equal(far[1], v)
    o, lse = fc.tree_attention(a, k, v, n, return_lse=True)
    assert torch.equal(o, fc.tree_attention(a, far[0], far[1], n))
    w = fc.attention_weight_sums(a, k, lse, causal=True, query_start=n, lengths=n + 5)
    assert torch.equal(w, fc.attention_weight_sums(a, far[0], lse, causal=True, query_start=n, lengths=n + 5))
    want = fc.evict_cache(k, v, w, n, 550)
    got = fc.evict_cache(far[0].clone(), far[1], w, n, 550)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    into = (torch.zeros(C << 22, dtype=torch.bfloat16, device="cuda").view(1, 1, C, 1 << 22)[..., :64], new(1, 1, C),
            torch.empty(1, 1, C, device="cuda"))
    got = fc.evict_cache(k, v, w, n, 550, out=into)
    assert torch.equal(got[0][:, :, :550], want[0]) and torch.equal(got[1][:, :, :550], want[1])


def test_in_inference_mode_and_what_autograd_knows(gpu_device):
    """The calls inside inference mode; and a graph that saved a cache which is written to afterwards refuses to run."""
    g = torch.Generator().manual_seed(4)
    new = lambda h, s: torch.randn(1, h, s, 64, generator=g).half().cuda()  # noqa: E731
    n = torch.tensor([20], dtype=torch.int32, device="cuda")
    f, _ = rot.rotary_frequencies(64, device="cuda")
    with torch.inference_mode():
        q, kc, vc = new(4, 3), new(2, 40), new(2, 40)
        q = fc.rotary_append(q, new(2, 3), new(2, 3), kc, vc, n, f)
        o, lse = fc.tree_attention(q, kc, vc, n, return_lse=True)
        w = fc.attention_weight_sums(q, kc, lse, causal=True, query_start=n, lengths=n + 3)
        fc.attention_weight_sums(q, kc, lse, causal=True, query_start=n, lengths=n + 3, into=w)
        fc.evict_cache(kc, vc, w, n + 3, 10, out=(new(2, 12), new(2, 12), torch.empty(1, 2, 12, device="cuda")))
        rot.rotary_embedding(q, None, f)
        total = w.double().sum(-1).cpu()
    assert bool(((total - 12).abs() <= 12 * 2.0 ** -9).all())
    kc, vc, x = new(2, 40), new(2, 40), new(2, 40).requires_grad_()
    y = (x * kc).sum()
    with torch.no_grad():
        fc.rotary_append(new(4, 1), new(2, 1), new(2, 1), kc, vc, n, f)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
