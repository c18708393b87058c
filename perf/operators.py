"""The operators around a K/V cache that this library is timed on: rotary positions, writing new tokens into a cache,
attention of a tree of drafted tokens over it, the attention weight its keys have received, and eviction by that weight.

``own = False`` computes each operator in its plain form, elementary torch operations in 32 bits (angles in 64);
``own = True`` calls the library.  ``exact`` is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# op: "rotary" (forward and gradients), "append", "tree", "weights", "evict".
# S: new tokens per sequence (drafted tokens, query rows); C: rows of the cache (keys); ragged: how much shorter the
# last sequence of a batch is than the first; rotary: rotated elements of a head; scaled: frequencies blended for long
# contexts; start: position of the first token; layout: storage order of the new tokens; branch: a tree's mean number
# of children (0: a chain without a mask); keep, recent, sinks: eviction's budget and what it never takes.
FIELDS = dict(op="rotary", dtype="bf16", B=1, Hq=32, Hkv=8, S=1, C=0, D=128, rotary=0, interleaved=False, scaled=False,
              start=0, layout="bnsd", ragged=0.0, branch=0, batch_trees=False, window=0, soft_cap=0.0, scale=0.0,
              spread=1.0, causal=False, keep=0, recent=0, sinks=0)


def case(name=None, **kw):
    assert not set(kw) - set(FIELDS), kw
    c = dict(FIELDS, **kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # Training a grouped-query layer of the benchmark's default shape: q and k rotated, and their gradients.
        case("rotary_train_gqa_s4096", op="rotary", dtype="bf16", B=2, S=4096, rotary=128),
        # Full-precision fine-tuning: part of the head, neighbouring pairs, frequencies scaled, far positions, odd length.
        case("rotary_train_fp32_part", op="rotary", dtype="fp32", Hq=8, Hkv=2, S=1000, rotary=64, interleaved=True,
             scaled=True, start=100000),
        # One new token of each sequence of a batch enters the cache: launches and host work count.
        case("append_decode_b8", op="append", dtype="bf16", B=8, S=1, C=4096, rotary=128, ragged=0.5),
        # A chunk of a prompt enters the cache, heads innermost as the projection writes them, odd length.
        case("append_chunk_s777", op="append", dtype="fp16", B=4, Hq=28, Hkv=4, S=777, C=8192, D=64, rotary=64,
             interleaved=True, layout="bsnd", ragged=0.3),
        # A small tree of one sequence over a short cache: latency.
        case("tree_t8_b1_4k", op="tree", dtype="bf16", S=8, C=4097, branch=2),
        # A batch with long caches of unequal lengths: memory-bound.
        case("tree_t16_b8_32k", op="tree", dtype="bf16", B=8, S=16, C=32768, branch=2, ragged=0.25),
        # Head dim 256, sliding window, soft-cap and its own scale, each sequence with a tree of its own.
        case("tree_gemma2_d256_8k", op="tree", dtype="bf16", B=2, Hq=16, Hkv=8, S=16, C=8192, D=256, branch=2,
             batch_trees=True, window=4096, soft_cap=50.0, scale=1.0 / 16, spread=2.0, ragged=0.4),
        # A wide tree, seven query heads per KV head: 448 rows share a KV head's cache, arithmetic counts.
        case("tree_t64_d64_16k", op="tree", dtype="fp16", B=4, Hq=28, Hkv=4, S=64, C=16384, D=64, branch=3, ragged=0.2),
        # The weight every prompt token received in a causal prefill of the benchmark's default shape: arithmetic.
        case("weights_prefill_gqa_s4096", op="weights", dtype="bf16", B=2, S=4096, C=4096, causal=True),
        # The same from the last 32 rows of a long prompt only.
        case("weights_last32_d64_16k", op="weights", dtype="fp16", B=4, Hq=28, Hkv=4, S=32, C=16383, D=64, causal=True),
        # A batch of prompts cut to a quarter of their length.
        case("evict_b8_8k", op="evict", dtype="bf16", B=8, Hkv=8, C=8192, keep=2048, recent=64, sinks=4, ragged=0.3),
        # One sequence of a small model, cut by half: latency.
        case("evict_b1_d64_2k", op="evict", dtype="fp32", Hkv=2, C=2048, D=64, keep=1000, recent=33, ragged=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, d):
    """(Hq, Hkv) of a layer."""
    return rng.choice([(16, 8), (16, 16), (8, 1)] if d == 256 else [(32, 8), (32, 32), (28, 4), (8, 2), (16, 2)])


def draw(rng):
    """One more case of the listed ranges: sizes spread over their logarithm, odd ones included."""
    op = rng.choice(["rotary", "append", "tree", "tree", "weights", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    es = BYTES[dtype]
    d = rng.choice([64, 128, 128, 256] if op != "evict" else [32, 64, 128, 128, 256])
    hq, hkv = _heads(rng, d)
    c = dict(op=op, dtype=dtype, D=d, Hq=hq, Hkv=hkv, layout=rng.choice(["bnsd", "bsnd"]))
    rot = dict(rotary=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5)
    if op == "rotary":
        most = 2 * 4096 * (32 + 8) * 128 * 2 // ((hq + hkv) * d * es)  # tokens of the largest listed case's bytes
        s = min(_log_int(rng, 64, 8192), most)
        return case(B=min(rng.randint(1, 4), most // s), S=s, start=rng.choice([0, 0, 1000, 100000]), **rot, **c)
    if op == "append":
        s = rng.choice([1, 1, _log_int(rng, 2, 1500)])
        b = rng.randint(1, 16) if s == 1 else rng.randint(1, 4)
        return case(B=b, S=s, C=s + _log_int(rng, 64, 8192), ragged=rng.uniform(0.0, 0.9), **rot, **c)
    if op == "tree":
        s = _log_int(rng, 1, 64)
        room = 7 * 8 * 32768 * 128 * 2 // (hkv * d * es)  # cache rows of about the largest listed case's bytes
        n = min(s + _log_int(rng, 64, 32768), room)
        most = room // n
        # (a row of the widest case costs what its keys cost to read)
        most = max(1, min(most, 4 * 28 * 64 * 16384 * 64 * 3 // (hq * s * n * d * (8 if dtype == "fp32" else 1))))
        gemma = d == 256
        return case(B=min(rng.randint(1, 8), most), S=s, C=n, ragged=rng.uniform(0.0, 0.9), branch=rng.choice([0, 2, 3]),
                    batch_trees=rng.random() < 0.5, window=rng.choice([0, 512, 4096]) if gemma else 0,
                    soft_cap=50.0 if gemma else rng.choice([0.0, 0.0, 30.0]), scale=1.0 / 16 if gemma else 0.0,
                    spread=2.0 if gemma else 1.0, **c)
    if op == "weights":
        kind = rng.choice(["prefill", "last", "decode"])
        if kind == "prefill":
            n = _log_int(rng, 128, 4096 if dtype != "fp32" else 1500)
            s, b = n, rng.randint(1, 2)
            if d == 256 or hq * d > 4096:
                b = 1
        else:
            n = _log_int(rng, 256, 20000)
            s, b = (1 if kind == "decode" else rng.randint(2, 64)), rng.randint(1, 4)
        return case(B=b, S=s, C=n, causal=kind != "decode", window=rng.choice([0, 0, 1000]) if kind == "prefill" else 0,
                    soft_cap=rng.choice([0.0, 0.0, 30.0]), ragged=rng.uniform(0.0, 0.9) if kind == "decode" else 0.0, **c)
    n = _log_int(rng, 128, 16384)
    keep = max(8, int(n * rng.uniform(0.1, 0.9)))
    most = max(1, 8 * 8 * 2048 * 128 * 2 // (hkv * keep * d * es))
    return case(B=min(rng.randint(1, 8), most), C=n, keep=keep, recent=rng.randint(0, keep // 2), sinks=rng.choice([0, 1, 4]),
                ragged=rng.uniform(0.0, 0.6), **c)


def _lengths(c):
    """Cached tokens of each sequence: the cache's rows less the new ones for the first, fewer for the later ones."""
    room = c["C"] - (c["S"] if c["op"] in ("append", "tree") else 0)
    return [max(1, round(room * (1.0 - c["ragged"] * b / max(1, c["B"] - 1)))) for b in range(c["B"])]


def _scale(c):
    return c["scale"] if c["scale"] else 1.0 / math.sqrt(c["D"])


def _inv_freq(c):
    """The angle of one position for each rotated pair, and the magnitude that goes with it, in 64 bits."""
    r, base = c["rotary"], 500000.0 if c["scaled"] else 10000.0
    i = torch.arange(0, r, 2, dtype=torch.float64)
    f = base ** (-i / r)
    if not c["scaled"]:
        return f, 1.0
    # four times the context the frequencies were made for: slow pairs interpolated, fast ones kept, a ramp between
    factor, length = 4.0, 8192
    turns = length * f / (2.0 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0


def _tree(c, g):
    """Which drafted tokens each of them sees ([trees, S, S], itself and its ancestors) and how deep it is."""
    masks, depths = [], []
    for _ in range(c["B"] if c["batch_trees"] else 1):
        seen, depth = torch.zeros(c["S"], c["S"], dtype=torch.bool), []
        pick = torch.rand(c["S"], generator=g).tolist()
        for t in range(c["S"]):
            last = (t - 1) // max(1, c["branch"])
            parent = t - 1 if c["branch"] == 0 else min(t - 1, max(-1, last - 1 + int(3 * pick[t])))
            if parent >= 0:
                seen[t] = seen[parent]
            seen[t, t] = True
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
        masks.append(seen)
        depths.append(depth)
    return torch.stack(masks), torch.tensor(depths, dtype=torch.int32)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def rand(h, s, spread=1.0, order="bnsd"):
        if order == "bsnd":
            return (torch.randn(c["B"], s, h, c["D"], generator=g, device=DEVICE) * spread).to(dtype).transpose(1, 2)
        return (torch.randn(c["B"], h, s, c["D"], generator=g, device=DEVICE) * spread).to(dtype)

    st = dict(case=c)
    op = c["op"]
    if op in ("rotary", "append"):
        st["q"], st["k"] = (rand(h, c["S"], order=c["layout"]) for h in (c["Hq"], c["Hkv"]))
        f, st["magnitude"] = _inv_freq(c)
        st["inv_freq"] = f.to(DEVICE)
    if op == "rotary":
        st["gq"], st["gk"] = (rand(h, c["S"], order=c["layout"]) for h in (c["Hq"], c["Hkv"]))
        st["q"].requires_grad_()
        st["k"].requires_grad_()
        st["positions"] = torch.arange(c["start"], c["start"] + c["S"], device=DEVICE)
        return st
    st["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEVICE)
    if op == "append":
        st["v"] = rand(c["Hkv"], c["S"], order=c["layout"])
        st["kc"], st["vc"] = rand(c["Hkv"], c["C"]), rand(c["Hkv"], c["C"])
        return st
    if op == "tree":
        st["q"] = rand(c["Hq"], c["S"], c["spread"], c["layout"])
        st["kc"], st["vc"] = rand(c["Hkv"], c["C"], c["spread"]), rand(c["Hkv"], c["C"])
        mask, depths = _tree(c, torch.Generator().manual_seed(seed))
        st["mask"] = mask.to(DEVICE) if c["branch"] else None
        st["depths"] = depths.expand(c["B"], c["S"]).contiguous().to(DEVICE)
        return st
    if op == "weights":
        st["q"], st["k"] = rand(c["Hq"], c["S"], order=c["layout"]), rand(c["Hkv"], c["C"], order=c["layout"])
        st["lse"] = torch.cat([torch.logsumexp(_weight_scores(c, st, b, torch.float32), dim=-1)
                               for b in range(c["B"])]).reshape(c["B"], c["Hq"], c["S"])
        return st
    st["kc"], st["vc"] = rand(c["Hkv"], c["C"]), rand(c["Hkv"], c["C"])
    # attention weight is concentrated: few keys hold most of it, and some none at all
    w = torch.exp(2.0 * torch.randn(c["B"], c["Hkv"], c["C"], generator=g, device=DEVICE))
    st["scores"] = torch.where(torch.rand(w.shape, generator=g, device=DEVICE) < 0.05, torch.zeros_like(w), w)
    return st


# ------------------------------------------------------------------------------------------------------ plain forms --
def _rotate(x, cos, sin, r, interleaved):
    """x [B, H, S, D] in 32 bits rotated by the angles of cos / sin [B, 1, S, r / 2]."""
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return y


def _angles(st, positions):
    """cos and sin of every (token, pair), the angles in 64 bits."""
    a = positions.to(torch.float64)[:, None, :, None] * st["inv_freq"]
    return (a.cos() * st["magnitude"]).float(), (a.sin() * st["magnitude"]).float()


def _plain_rotary(c, st):
    cos, sin = _angles(st, st["positions"][None])
    turn = lambda x, s: _rotate(x.detach().float(), cos, s, c["rotary"], c["interleaved"]).to(x.dtype)  # noqa: E731
    return [turn(st["q"], sin), turn(st["k"], sin), turn(st["gq"], -sin), turn(st["gk"], -sin)]


def _plain_append(c, st):
    pos = st["lengths"][:, None] + torch.arange(c["S"], device=DEVICE)
    cos, sin = _angles(st, pos)
    q = _rotate(st["q"].float(), cos, sin, c["rotary"], c["interleaved"]).to(st["q"].dtype)
    k = _rotate(st["k"].float(), cos, sin, c["rotary"], c["interleaved"]).to(st["k"].dtype)
    b = torch.arange(c["B"], device=DEVICE)[:, None]
    st["kc"][b, :, pos] = k.transpose(1, 2)
    st["vc"][b, :, pos] = st["v"].transpose(1, 2)
    return [q, st["kc"], st["vc"]]


def _tree_allowed(c, st):
    """[B, S, C]: which cache rows each drafted token sees."""
    j = torch.arange(c["C"], device=DEVICE)
    n = st["lengths"].long()[:, None]
    cached = (j < n)[:, None, :].expand(c["B"], c["S"], c["C"])
    if c["window"]:
        cached = cached & ((n + st["depths"])[..., None] - j <= c["window"])
    u = (j - n).clamp(0, c["S"] - 1)
    mask = st["mask"] if st["mask"] is not None else torch.ones(1, c["S"], c["S"], dtype=torch.bool, device=DEVICE).tril()
    own_tree = mask.expand(c["B"], -1, -1).gather(2, u[:, None, :].expand(c["B"], c["S"], c["C"]))
    return cached | (own_tree & ((j >= n) & (j < n + c["S"]))[:, None, :])


def _plain_tree(c, st):
    B, G, S, D = c["B"], c["Hq"] // c["Hkv"], c["S"], c["D"]
    q = st["q"].float().reshape(B, c["Hkv"], G * S, D)
    x = torch.matmul(q, st["kc"].float().transpose(2, 3)) * _scale(c)
    if c["soft_cap"]:
        x = c["soft_cap"] * torch.tanh(x / c["soft_cap"])
    x = x.view(B, c["Hkv"], G, S, c["C"]).masked_fill(~_tree_allowed(c, st)[:, None, None], float("-inf"))
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul((p / total).view(B, c["Hkv"], G * S, c["C"]), st["vc"].float())
    lse = (m + torch.log(total)).reshape(B, c["Hq"], S)
    return [o.view(B, c["Hq"], S, D).to(st["q"].dtype), lse]


def _weight_scores(c, st, b, dtype):
    """The masked scores of sequence b in ``dtype``: [Hkv, G * S, C]."""
    q = st["q"][b].to(dtype).reshape(c["Hkv"], -1, c["D"])
    x = torch.matmul(q, st["k"][b].to(dtype).transpose(1, 2)) * _scale(c)
    if c["soft_cap"]:
        x = c["soft_cap"] * torch.tanh(x / c["soft_cap"])
    j = torch.arange(c["C"], device=x.device)
    i = torch.arange(c["C"] - c["S"], c["C"], device=x.device)[:, None]
    ok = (j < st["lengths"][b].to(x.device)).expand(c["S"], c["C"])
    if c["causal"]:
        ok = ok & (j <= i)
    if c["window"]:
        ok = ok & (i - j <= c["window"])
    return x.view(c["Hkv"], -1, c["S"], c["C"]).masked_fill(~ok, float("-inf"))


def _plain_weights(c, st):
    G = c["Hq"] // c["Hkv"]
    q = st["q"].float().reshape(c["B"], c["Hkv"], G * c["S"], c["D"])
    x = torch.matmul(q, st["k"].float().transpose(2, 3)) * _scale(c)
    if c["soft_cap"]:
        x = c["soft_cap"] * torch.tanh(x / c["soft_cap"])
    j = torch.arange(c["C"], device=DEVICE)
    i = torch.arange(c["C"] - c["S"], c["C"], device=DEVICE)[:, None]
    ok = (j < st["lengths"][:, None, None]).expand(c["B"], c["S"], c["C"])
    if c["causal"]:
        ok = ok & (j <= i)
    if c["window"]:
        ok = ok & (i - j <= c["window"])
    x = x.view(c["B"], c["Hkv"], G, c["S"], c["C"]).masked_fill(~ok[:, None, None], float("-inf"))
    return torch.exp(x - st["lse"].view(c["B"], c["Hkv"], G, c["S"], 1)).sum(dim=(2, 3))


def _plain_evict(c, st):
    n, keep = st["lengths"].long()[:, None, None], c["keep"]
    j = torch.arange(c["C"], device=DEVICE)
    # the order of going: rows behind the length first, then by weight, never the first and the last ones
    rank = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), 2, 1)
    rank = torch.where(j < n, rank, 0).expand(c["B"], c["Hkv"], c["C"])
    order = torch.argsort(st["scores"], dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(rank.gather(-1, order), dim=-1, descending=True, stable=True))
    slots = order[..., :keep].where(torch.arange(keep, device=DEVICE) < n, c["C"]).sort(dim=-1).values
    live = slots < c["C"]
    at = slots.clamp(max=c["C"] - 1)
    row = at[..., None].expand(-1, -1, -1, c["D"])
    none = ~live[..., None]
    return [st["kc"].gather(2, row).masked_fill(none, 0), st["vc"].gather(2, row).masked_fill(none, 0),
            st["scores"].gather(2, at).masked_fill(~live, 0), slots.masked_fill(~live, -1).int(),
            st["lengths"].clamp(max=keep)]


# ------------------------------------------------------------------------------------------------------------- runs --
def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu-flex-att_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flexatt_cache
    import flexatt_rotary

    return flexatt_rotary, flexatt_cache


def _own_run(c, st):
    rotary, cache = _library()
    op = c["op"]
    if op == "rotary":
        out = rotary.rotary_embedding(st["q"], st["k"], st["inv_freq"], positions=st["positions"],
                                      interleaved=c["interleaved"], magnitude=st["magnitude"])
        grads = torch.autograd.grad(out, (st["q"], st["k"]), (st["gq"], st["gk"]))
        return [out[0].detach(), out[1].detach(), grads[0], grads[1]]
    if op == "append":
        q = cache.rotary_append(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["lengths"], st["inv_freq"],
                                interleaved=c["interleaved"], magnitude=st["magnitude"])
        return [q, st["kc"], st["vc"]]
    if op == "tree":
        return list(cache.tree_attention(st["q"], st["kc"], st["vc"], st["lengths"], st["mask"],
                                         sliding_window=c["window"], depths=st["depths"], scale=_scale(c),
                                         soft_cap=c["soft_cap"], return_lse=True))
    if op == "weights":
        return cache.attention_weight_sums(st["q"], st["k"], st["lse"], causal=c["causal"],
                                           query_start=c["C"] - c["S"], lengths=st["lengths"],
                                           sliding_window=c["window"], scale=_scale(c), soft_cap=c["soft_cap"])
    return list(cache.evict_cache(st["kc"], st["vc"], st["scores"], st["lengths"], c["keep"], recent=c["recent"],
                                  sinks=c["sinks"]))


PLAIN = dict(rotary=_plain_rotary, append=_plain_append, tree=_plain_tree, weights=_plain_weights, evict=_plain_evict)


def run(st):
    c = st["case"]
    if own:
        return _own_run(c, st)
    with torch.no_grad():
        return PLAIN[c["op"]](c, st)


def _causal_pairs(c):
    """(row, key) pairs of one head that the masks of a weights case leave."""
    if not c["causal"]:
        return sum(_lengths(c)) * c["S"]
    most = c["window"] + 1 if c["window"] else c["C"]
    return c["B"] * sum(min(i + 1, most) for i in range(c["C"] - c["S"], c["C"]))


def work(c):
    """Each input read once and each output written once; the pairs that the masks leave."""
    es, op = BYTES[c["dtype"]], c["op"]
    new_q, new_k = (c["B"] * h * c["S"] * c["D"] * es for h in (c["Hq"], c["Hkv"]))
    if op == "rotary":
        pairs = c["B"] * (c["Hq"] + c["Hkv"]) * c["S"] * c["rotary"] // 2
        return {"bytes": 4 * (new_q + new_k) + 8 * c["S"] + 4 * c["rotary"], "flops": 12 * pairs}
    if op == "append":
        pairs = c["B"] * (c["Hq"] + c["Hkv"]) * c["S"] * c["rotary"] // 2
        return {"bytes": 2 * (new_q + 2 * new_k) + 4 * c["B"] + 4 * c["rotary"], "flops": 6 * pairs}
    if op == "tree":
        # a window leaves a tree's first token its width of cached keys
        cached = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        rows = cached + c["B"] * c["S"]
        pairs = c["Hq"] * (cached * c["S"] + c["B"] * c["S"] * (c["S"] + 1) // 2)
        return {"bytes": 2 * new_q + 2 * rows * c["Hkv"] * c["D"] * es + 4 * c["B"] * c["Hq"] * c["S"],
                "flops": 4 * c["D"] * pairs}
    if op == "weights":
        keys = sum(_lengths(c)) * c["Hkv"] * c["D"] * es
        return {"bytes": new_q + keys + 4 * c["B"] * (c["Hq"] * c["S"] + c["Hkv"] * c["C"]),
                "flops": 2 * c["D"] * c["Hq"] * _causal_pairs(c)}
    kept = sum(min(n, c["keep"]) for n in _lengths(c)) * c["Hkv"]
    return {"bytes": kept * (4 * c["D"] * es + 12) + 4 * c["Hkv"] * sum(_lengths(c)), "flops": 0}


# ------------------------------------------------------------------------------------------------------------ exact --
def exact(c, seed):
    """The definitions in 64 bits, on the CPU or (attention's large products) on the GPU; one sequence or head at a time."""
    st = prepare(c, seed)
    op = c["op"]
    wide = lambda x: x.detach().double()  # noqa: E731
    if op in ("rotary", "append"):
        lengths = _lengths(c) if op == "append" else None
        r = c["rotary"]
        first, second = (range(0, r, 2), range(1, r, 2)) if c["interleaved"] else (range(r // 2), range(r // 2, r))
        first, second = torch.tensor(first, device=DEVICE), torch.tensor(second, device=DEVICE)

        def turned(x, back):
            y = wide(x)
            for b in range(c["B"]):
                p = torch.arange(c["S"], dtype=torch.float64, device=DEVICE) + (lengths[b] if lengths else c["start"])
                z = torch.polar(torch.full((c["S"], r // 2), st["magnitude"], dtype=torch.float64, device=DEVICE),
                                torch.outer(p, st["inv_freq"]) * (-1.0 if back else 1.0))
                w = torch.complex(y[b].index_select(-1, first), y[b].index_select(-1, second)) * z
                y[b].index_copy_(-1, first, w.real)
                y[b].index_copy_(-1, second, w.imag)
            return y

        if op == "rotary":
            return [turned(st["q"], False), turned(st["k"], False), turned(st["gq"], True), turned(st["gk"], True)]
        kc, vc, k = wide(st["kc"]), wide(st["vc"]), turned(st["k"], False)
        for b, n in enumerate(lengths):
            kc[b, :, n:n + c["S"]] = k[b]
            vc[b, :, n:n + c["S"]] = wide(st["v"][b])
        return [turned(st["q"], False), kc, vc]
    G = c["Hq"] // c["Hkv"]
    if op == "tree":
        o = torch.empty(c["B"], c["Hq"], c["S"], c["D"], dtype=torch.float64, device=DEVICE)
        lse = torch.empty(c["B"], c["Hq"], c["S"], dtype=torch.float64, device=DEVICE)
        depths = st["depths"].long()
        for b, n in enumerate(_lengths(c)):
            seen = (torch.ones(c["S"], c["S"], dtype=torch.bool, device=DEVICE).tril() if st["mask"] is None
                    else st["mask"][b % st["mask"].shape[0]])
            head = torch.ones(c["S"], n, dtype=torch.bool, device=DEVICE)
            if c["window"]:
                head = torch.arange(n, device=DEVICE)[None, :] >= (n + depths[b] - c["window"])[:, None]
            hidden = ~torch.cat((head, seen), dim=1)
            for h in range(c["Hq"]):
                k, v = (wide(st[x][b, h // G, :n + c["S"]]) for x in ("kc", "vc"))
                x = wide(st["q"][b, h]) @ k.T * _scale(c)
                if c["soft_cap"]:
                    x = torch.tanh(x / c["soft_cap"]) * c["soft_cap"]
                x[hidden] = float("-inf")
                lse[b, h] = torch.logsumexp(x, dim=1)
                o[b, h] = torch.softmax(x, dim=1) @ v
        return [o, lse]
    if op == "weights":
        w = torch.zeros(c["B"], c["Hkv"], c["C"], dtype=torch.float64, device=DEVICE)
        at = torch.arange(c["C"] - c["S"], c["C"], device=DEVICE)
        for b, n in enumerate(_lengths(c)):
            keys = torch.arange(n, device=DEVICE)
            far = at[:, None] - keys[None, :]
            hidden = (far < 0 if c["causal"] else torch.zeros_like(far, dtype=torch.bool))
            if c["window"]:
                hidden = hidden | (far > c["window"])
            for h in range(c["Hq"]):
                x = wide(st["q"][b, h]) @ wide(st["k"][b, h // G, :n]).T * _scale(c)
                if c["soft_cap"]:
                    x = torch.tanh(x / c["soft_cap"]) * c["soft_cap"]
                x -= wide(st["lse"][b, h])[:, None]
                x[hidden] = float("-inf")
                w[b, h // G, :n] += x.exp().sum(dim=0)
        return w
    # eviction: a sort of each head's slots on the host, then plain copies
    keep, scores = c["keep"], st["scores"].cpu()
    out = [torch.zeros(c["B"], c["Hkv"], keep, c["D"], dtype=torch.float64, device=DEVICE) for _ in range(2)]
    kept = torch.zeros(c["B"], c["Hkv"], keep, dtype=torch.float64)
    slots = torch.full((c["B"], c["Hkv"], keep), -1, dtype=torch.int32)
    for b, n in enumerate(_lengths(c)):
        for h in range(c["Hkv"]):
            w = scores[b, h, :n].tolist()
            free = range(min(c["sinks"], n), max(n - c["recent"], min(c["sinks"], n)))
            best = set(sorted(free, key=lambda j: (-w[j], j))[:max(0, keep - (n - len(free)))])
            stay = torch.tensor([j for j in range(n) if j not in free or j in best][:keep])
            slots[b, h, :len(stay)] = stay.int()
            kept[b, h, :len(stay)] = scores[b, h, stay].double()
            for x, y in zip(out, (st["kc"], st["vc"])):
                x[b, h, :len(stay)] = wide(y[b, h, stay.to(DEVICE)])
    return out + [kept, slots, torch.tensor([min(n, keep) for n in _lengths(c)], dtype=torch.int32)]
