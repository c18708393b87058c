"""Norm and rotation, caches of 8 bits and shared prefixes one after the other, as training and a server use them, each
step held against the float64 oracle on the GPU's own inputs of that step; and calls that no test of one operator makes."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

import flexatt_cache as fc
import flexatt_rotary as rot
import npu_flash_attention as nfa
from gpu_helpers import TOL, err
from oracle import attention_oracle as aorc
from oracle import cache_oracle as orc
from test_gpu_norm_rotary import weight
from test_gpu_quant_cache import bits
from test_gpu_quant_tree import cache
from test_gpu_tree import check, draw, tree

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
F8, I8 = torch.float8_e4m3fn, torch.int8


def near(x, ref, tol, what):
    worst = ((x.cpu().double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} tolerances"


def empty(B, H, C, D, kind):
    c = [torch.zeros(B, H, C, D, dtype=torch.uint8, device="cuda").view(kind) for _ in range(2)]
    return c + [torch.zeros(B, H, C, device="cuda") for _ in range(2)]


def host(*xs):
    return [x.cpu() for x in xs]


def ints(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,kind,D,inter", [(BF, F8, 128, False), (FH, I8, 64, True)])
def test_prompt_in_chunks_then_drafts(gpu_device, dtype, kind, D, inter):
    """A prompt is normalised, turned, written to a cache of 8 bits and attended, a second chunk of it behind the cached
    one read back, then drafted tokens over the cache; the accepted ones stay."""
    B, Hq, Hkv, S, S2, T, room = 2, 8, 2, 150, 61, 7, 260
    wq, wk = weight(1, D, dtype), weight(2, D, dtype)
    f, m = rot.rotary_frequencies(D, scaling="yarn", factor=4.0, original_length=64, device="cuda")
    kw = dict(interleaved=inter, magnitude=m)
    store = empty(B, Hkv, room, D, kind)
    n = ints(0, 0)

    def new(seed, s):
        return draw(seed, B, Hq, s, D, dtype, "bsnd"), draw(seed + 1, B, Hkv, s, D, dtype, "bsnd"), draw(seed + 2, B, Hkv, s, D, dtype)

    # the first chunk, attended in the working type; what the append returns are the same queries
    q, k, v = new(10, S)
    yq, yk = rot.norm_rotary_embedding(q, k, wq, wk, f, **kw)
    assert torch.equal(fc.quantized_append(q, k, v, *store, n, f, query_weight=wq, key_weight=wk, **kw), yq)
    o, lse = nfa.npu_flash_attention_forward(yq, yk, v, causal=True, return_lse=True)
    ro, rl = aorc.forward(*host(yq, yk, v), True)
    assert err(o, ro) <= TOL[dtype]["o"] and err(lse, rl) <= TOL[dtype]["lse"]
    n += S

    # the second chunk, behind what the cache gives back
    q, k, v = new(20, S2)
    yq = fc.quantized_append(q, k, v, *store, n, f, query_weight=wq, key_weight=wk, **kw)
    n += S2
    bk, bv = fc.dequantize_cache(*store, n, dtype=dtype)
    rows = S + S2
    back = bits(store[0]).view(kind).float().double() * store[2].double()[..., None]
    assert torch.equal(bk[:, :, :rows], back.float().to(dtype)[:, :, :rows]) and bool((bk[:, :, rows:] == 0).all())
    o, lse = nfa.npu_flash_attention_forward(yq, bk[:, :, :rows], bv[:, :, :rows], causal=True, return_lse=True)
    a, la = fc.quantized_tree_attention(yq, *store, n - S2, return_lse=True)  # the chunk as drafted tokens: the same keys
    ro, rl, to, tl = orc.quantized_tree_attention(*host(yq, *store, n - S2), dtype=dtype)
    check("o", a, ro, to)
    check("lse", la, rl, tl)
    ro, rl = aorc.forward(*host(yq, bk[:, :, :rows], bv[:, :, :rows]), True)  # (its causal mask counts from the first key)
    assert err(o, ro) <= TOL[dtype]["o"] and err(lse, rl) <= TOL[dtype]["lse"]

    # drafted tokens, a tree
    mask, depth = tree(T, 3, "shared")
    q, k, v = new(30, T)
    pos = n[:, None] + depth.cuda()
    yq = fc.quantized_append(q, k, v, *store, n, f, positions=pos, query_weight=wq, key_weight=wk, **kw)
    ref, slack = orc.norm_rotary(q.cpu().double(), wq.cpu().double(), f.cpu(), pos.cpu(), inter, m)
    near(yq, ref, orc.rounded(ref, slack, dtype), "q")
    for window in (0, 40):
        a, la = fc.quantized_tree_attention(yq, *store, n, mask.cuda(), sliding_window=window,
                                            depths=depth.cuda() if window else None, return_lse=True)
        ro, rl, to, tl = orc.quantized_tree_attention(*host(yq, *store, n), mask, window, depth.expand(B, T), dtype=dtype)
        check("o", a, ro, to)
        check("lse", la, rl, tl)

    # the first token is accepted: its row stays, the next step is one token per sequence
    n += 1
    q, k, v = new(40, 1)
    yq = fc.quantized_append(q, k, v, *store, n, f, query_weight=wq, key_weight=wk, **kw)
    a, la = fc.quantized_tree_attention(yq, *store, n, return_lse=True)
    ro, rl, to, tl = orc.quantized_tree_attention(*host(yq, *store, n), dtype=dtype)
    check("o", a, ro, to)
    check("lse", la, rl, tl)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FS, 64)])
def test_behind_a_shared_prompt(gpu_device, dtype, D):
    """A shared prompt normalised and turned once, continuations of unequal length appended behind it, drafted tokens
    attended: what every sequence gets alone from a cache that holds both."""
    B, Hq, Hkv, P, S, T = 5, 4, 2, 300, 33, 3
    wq, wk = weight(1, D, FS), weight(2, D, FS)
    f, _ = rot.rotary_frequencies(D, device="cuda")
    pk, pv = draw(1, 1, Hkv, P, D, dtype), draw(2, 1, Hkv, P, D, dtype)
    _, pk = rot.norm_rotary_embedding(draw(3, 1, Hq, P, D, dtype), pk, wq, wk, f)
    kc, vc = draw(4, B, Hkv, 80, D, dtype), draw(5, B, Hkv, 80, D, dtype)
    n = ints(0, 1, 33, 20, 7)
    zero = torch.zeros_like(n)
    pos = P + torch.arange(S, device="cuda")
    fc.norm_rotary_append(draw(6, B, 0, S, D, dtype), draw(7, B, Hkv, S, D, dtype), draw(8, B, Hkv, S, D, dtype), kc, vc, zero,
                          wq, wk, f, positions=pos)
    q, k, v = draw(9, B, Hq, T, D, dtype), draw(10, B, Hkv, T, D, dtype), draw(11, B, Hkv, T, D, dtype)
    yq = fc.norm_rotary_append(q, k, v, kc, vc, n, wq, wk, f, positions=P + n[:, None] + torch.arange(T, device="cuda"))
    alone = torch.cat((pk.expand(B, -1, -1, -1), kc), 2), torch.cat((pv.expand(B, -1, -1, -1), vc), 2)
    for window in (0, 50):
        o, lse = fc.shared_prefix_attention(yq, pk[0], pv[0], kc, vc, n, sliding_window=window, return_lse=True)
        ro, rl, to, tl = orc.prefix_attention(*host(yq, pk[0], pv[0], kc, vc, n), window=window, dtype=dtype)
        check("o", o, ro, to)
        check("lse", lse, rl, tl)
        a, la = fc.tree_attention(yq, *alone, P + n, sliding_window=window, return_lse=True)
        near(a, ro, to, "o alone")
        near(la, rl, tl, "lse alone")
    want = orc.norm_rotary(k.cpu().double(), wk.cpu().double(), f.cpu(), (P + n[:, None] + torch.arange(T, device="cuda")).cpu())
    for b, x in enumerate(n.tolist()):
        near(kc[b, :, x:x + T], want[0][b], orc.rounded(*want, dtype)[b], "k")


def test_a_training_step(gpu_device):
    """Norm, rotation and attention forward and back: the gradients of a layer's queries, keys and weights."""
    B, Hq, Hkv, S, D = 2, 4, 2, 70, 64
    q, k, v = draw(1, B, Hq, S, D, FS), draw(2, B, Hkv, S, D, FS), draw(3, B, Hkv, S, D, FS)
    wq, wk, f = weight(4, D, FS), weight(5, D, FS), rot.rotary_frequencies(D, device="cuda")[0]
    g = draw(6, B, Hq, S, D, FS)
    leaves = [x.requires_grad_() for x in (q, k, v, wq, wk)]
    y, z = rot.norm_rotary_embedding(q, k, wq, wk, f)
    got = torch.autograd.grad(nfa.npu_flex_attention(y, z, v, causal=True), leaves, g)
    a, b, c, d, e = (x.detach().cpu().double().requires_grad_() for x in leaves)
    pos = torch.arange(S).expand(B, S)
    x = orc.norm_rotary(a, d, f.cpu(), pos)[0] @ orc.norm_rotary(b, e, f.cpu(), pos)[0].repeat_interleave(2, 1).transpose(2, 3)
    x = (x / D ** 0.5).masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
    want = torch.autograd.grad(x.softmax(-1) @ c.repeat_interleave(2, 1), (a, b, c, d, e), g.cpu().double())
    for x, r, what in zip(got, want, ("dq", "dk", "dv", "dq", "dk")):
        assert err(x, r) <= TOL[FS][what]


def test_values_of_very_unequal_scales(gpu_device):
    """A value whose scale is 2^17 times the others', and whose weight is as small: the others keep their bits.

    fp16 holds p s' to 2^-12 of itself from 2^-14 on and to 2^-25 under that, and the largest scale is at least 2^6 there:
    n 2^-31 times it over the row's sum of weights, in place of the oracle's n 2^-24."""
    n, D = 40, 64
    for dtype in (BF, FH):
        for kind in (F8, I8):
            (kc, ks), (vc, vs) = cache(1, 1, 1, n + 1, D, kind, 0.0), cache(2, 1, 1, n + 1, D, kind, 0.0)
            q = torch.ones(1, 1, 1, D, dtype=dtype, device="cuda")
            ks *= 0.02
            bits(kc)[0, 0, 17] = bits(torch.full((D,), -100.0 if kind == I8 else -96.0).to(kind)).cuda()
            ks[0, 0, 17] = 12.0 / (8 * 96)
            vs[0, 0, 17] *= 2.0 ** 17
            args = (q, kc, vc, ks, vs, ints(n))
            o, lse = fc.quantized_tree_attention(*args, return_lse=True)
            ro, rl, to, tl = orc.quantized_tree_attention(*host(*args), dtype=dtype)
            x = (q.double() @ (kc.float().double() * ks.double()[..., None]).transpose(2, 3)) / D ** 0.5
            total = torch.exp(x - x.max()).sum().item()
            floor = (n + 1) * vs.double().max().item() * orc.TOP[kind]
            v = (vc.float().double() * vs.double()[..., None])[0, 0].cpu()
            p = torch.exp(x - rl.cuda()[..., None])[0, 0, 0].cpu()
            # half a step of each weight, the scores' and sums' roundings as everywhere
            slack = (p[:, None] * v.abs()).sum(0) * (2.0 ** -12 + 2.0 ** -18) + floor * 2.0 ** -31 / total
            near(o[0, 0, 0], ro[0, 0, 0], orc.rounded(ro[0, 0, 0], slack, dtype), f"{dtype} {kind}")
            check("lse", lse, rl, tl)


def test_offsets_past_32_bits(gpu_device):
    """Rows 2^22 elements apart, so that row 520 of 8 bits and of 16 starts past 2^31 bytes: as from dense ones, bit for bit."""
    D, C, kind = 64, 600, I8
    wide = torch.zeros(C << 22, dtype=torch.int8, device="cuda").view(1, 1, C, 1 << 22)
    far = [wide[..., 64 * i:64 * i + 64] for i in range(2)]
    (kc, ks), (vc, vs) = cache(1, 1, 1, C, D, kind), cache(2, 1, 1, C, D, kind)
    far[0].copy_(kc), far[1].copy_(vc)
    n, f = ints(590), rot.rotary_frequencies(D, device="cuda")[0]
    q, k, v, w = draw(3, 1, 2, 5, D, BF), draw(4, 1, 1, 5, D, BF), draw(5, 1, 1, 5, D, BF), weight(6, D, BF)
    s = [ks.clone(), vs.clone()]
    a = fc.quantized_append(q, k, v, kc, vc, ks, vs, n, f, query_weight=w, key_weight=w)
    assert torch.equal(a, fc.quantized_append(q, k, v, *far, *s, n, f, query_weight=w, key_weight=w))
    assert torch.equal(far[0], kc) and torch.equal(far[1], vc) and torch.equal(s[0], ks) and torch.equal(s[1], vs)
    assert torch.equal(fc.quantized_tree_attention(a, kc, vc, ks, vs, n), fc.quantized_tree_attention(a, *far, ks, vs, n))
    x, y = fc.dequantize_cache(kc, vc, ks, vs, n), fc.dequantize_cache(*far, ks, vs, n)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    del wide, far
    wide = torch.zeros(C << 22, dtype=BF, device="cuda").view(1, C, 1 << 22)
    pk, pv = x[0][0], x[1][0]
    out = wide[..., 64:128][None], wide[..., 256:320][None]
    y = fc.dequantize_cache(kc, vc, ks, vs, n, out=out)
    assert y[0] is out[0] and torch.equal(out[0], x[0]) and torch.equal(out[1], x[1])
    own = draw(7, 1, 1, 20, D, BF)
    assert torch.equal(fc.shared_prefix_attention(q, out[0][0], out[1][0], own, own, ints(9)),
                       fc.shared_prefix_attention(q, pk, pv, own, own, ints(9)))
    k3, v3 = pk[None].clone(), pv[None].clone()
    b = fc.norm_rotary_append(q, k, v, k3, v3, n, w, w, f)
    assert torch.equal(b, fc.norm_rotary_append(q, k, v, *out, n, w, w, f)) and torch.equal(out[0], k3) and torch.equal(out[1], v3)


def test_scales_and_inputs_of_any_strides(gpu_device):
    """Scales that are not contiguous are read where they are only read; inputs that repeat one row or head."""
    (kc, ks), (vc, vs) = cache(1, 3, 2, 100, 64, F8), cache(2, 3, 2, 100, 64, F8)
    n, q = ints(99, 40, 0), draw(3, 3, 4, 1, 64, FH)
    odd = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (ks, vs)]
    assert not odd[0].is_contiguous()
    assert torch.equal(fc.quantized_tree_attention(q, kc, vc, *odd, n), fc.quantized_tree_attention(q, kc, vc, ks, vs, n))
    a, b = fc.dequantize_cache(kc, vc, *odd, n), fc.dequantize_cache(kc, vc, ks, vs, n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for s in (odd, (ks, odd[1])):
        with pytest.raises(RuntimeError, match="contiguous"):
            fc.quantized_append(q, q[:, :2], q[:, :2], kc, vc, *s, n, None)
    one = q[:1].expand(3, 4, 1, 64)  # one sequence's queries for all
    assert torch.equal(fc.quantized_tree_attention(one, kc, vc, ks, vs, n),
                       fc.quantized_tree_attention(one.contiguous(), kc, vc, ks, vs, n))
    k1 = kc[:, :1].expand(3, 2, 100, 64)  # one head's codes for both, read only
    assert torch.equal(fc.quantized_tree_attention(q, k1, vc, ks, vs, n),
                       fc.quantized_tree_attention(q, k1.contiguous(), vc, ks, vs, n))
    f, w = rot.rotary_frequencies(64, device="cuda")[0], weight(4, 64, FH)
    y = rot.norm_rotary_embedding(one, one, w, w, f, positions=ints(5).expand(1))
    z = rot.norm_rotary_embedding(one.contiguous(), one.contiguous(), w, w, f, positions=ints(5))
    assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])


def test_two_at_once(gpu_device):
    """Two calls of each on two streams, and two captured graphs replayed side by side, give what one alone gives."""
    sets = []
    for i in range(2):
        (kc, ks), (vc, vs) = cache(1 + i, 2, 2, 4000, 128, F8), cache(3 + i, 2, 2, 4000, 128, F8)
        sets.append((draw(5 + i, 2, 8, 4, 128, BF), kc, vc, ks, vs, ints(3900, 1000 + i)))
    k, v = draw(8, 2, 2, 50, 128, BF), draw(9, 2, 2, 50, 128, BF)
    pk, pv = draw(10, 1, 2, 3000, 128, BF)[0], draw(11, 1, 2, 3000, 128, BF)[0]

    def run(i):
        q = sets[i][0]
        return [fc.quantized_tree_attention(*sets[i]), fc.shared_prefix_attention(q, pk, pv, k, v, ints_of[i])]

    ints_of = [ints(40, 3), ints(7, 46)]
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for i in range(2):
            with torch.cuda.stream(sides[i]):
                got.append(run(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            outs.append(run(i))
    for turn in range(3):
        sets[turn % 2][0].copy_(draw(20 + turn, 2, 8, 4, 128, BF))
        for i in range(2):  # (graphs of one pool run one after the other)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip([x.clone() for x in outs[i]], run(i)))


def test_inference_mode_tangents_and_traces(gpu_device):
    (kc, ks), (vc, vs) = cache(1, 1, 2, 60, 64, I8), cache(2, 1, 2, 60, 64, I8)
    q, k = draw(3, 1, 4, 3, 64, FH), draw(4, 1, 2, 3, 64, FH)
    n, f, w = ints(20), rot.rotary_frequencies(64, device="cuda")[0], weight(5, 64, FH)
    own = draw(6, 1, 2, 60, 64, FH)
    calls = [lambda x: rot.norm_rotary_embedding(x, None, w, None, f)[0],
             lambda x: fc.norm_rotary_append(x, k, k, own.clone(), own.clone(), n, w, w, f),
             lambda x: fc.quantized_append(x, k, k, kc, vc, ks, vs, n, f, query_weight=w, key_weight=w),
             lambda x: fc.quantized_tree_attention(x, kc, vc, ks, vs, n),
             lambda x: fc.shared_prefix_attention(x, own[0], own[0], own, own, n)]
    for call in calls:
        plain = call(q)
        with torch.inference_mode():
            assert torch.equal(call(q), plain)
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                call(fwd.make_dual(q, torch.ones_like(q)))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(q[None])
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call)(q)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda s: fc.dequantize_cache(kc, vc, s, vs, n)[0])(ks)
    for call in calls[1:]:
        with pytest.raises(RuntimeError):
            call(q.clone().requires_grad_())
    x = q.clone().requires_grad_()
    y = rot.norm_rotary_embedding(x, None, w, None, f)[0]
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == q.shape
    y = rot.norm_rotary_embedding(x, None, w, None, f)[0]
    with torch.no_grad():
        x += 1  # what the gradient needs has changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_one_tensor_as_query_and_key(gpu_device):
    """The same leaf and the same weight twice: their gradients are the sums."""
    f = rot.rotary_frequencies(64, device="cuda")[0]
    x, w = draw(1, 1, 2, 9, 64, FS).requires_grad_(), weight(2, 64, FS).requires_grad_()
    g, h = draw(3, 1, 2, 9, 64, FS), draw(4, 1, 2, 9, 64, FS)
    y = rot.norm_rotary_embedding(x, x, w, w, f)
    dx, dw = torch.autograd.grad(y, (x, w), (g, h))
    pos = torch.arange(9)[None]
    (rx, sx), (rw, sw) = orc.norm_rotary_grad(*(t.detach().cpu().double() for t in (x, w, g)), f.cpu(), pos)
    (rx2, sx2), (rw2, sw2) = orc.norm_rotary_grad(*(t.detach().cpu().double() for t in (x, w, h)), f.cpu(), pos)
    near(dx, rx + rx2, orc.rounded(rx + rx2, sx + sx2, FS) + (rx.abs() + rx2.abs()) * 2.0 ** -23, "dx")
    near(dw, rw + rw2, orc.rounded(rw + rw2, sw + sw2, FS) + (rw.abs() + rw2.abs()) * 2.0 ** -23, "dw")


@pytest.mark.parametrize("T", [2047, 4096])
def test_many_drafted_tokens(gpu_device, T):
    """A prompt of its own as drafted tokens over a cache with nothing else: rows of every length, no mask."""
    (kc, ks), (vc, vs) = cache(1, 1, 1, T, 64, F8), cache(2, 1, 1, T, 64, F8)
    q = draw(3, 1, 1, T, 64, BF)
    o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, ints(0), return_lse=True)
    ro, rl, to, tl = orc.quantized_tree_attention(*host(q, kc, vc, ks, vs, ints(0)))
    check("o", o, ro, to)
    check("lse", lse, rl, tl)
