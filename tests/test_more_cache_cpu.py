"""Refusals of the norm's, the 8-bit cache's and its attention's entry points (Python and C ABI), and their oracle, on the
host.  No kernel is launched here."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_lib as L
import flexatt_rotary as rot
from oracle import cache_oracle as orc

FAKE = 1 << 20  # aligned, never dereferenced: every call below fails its checks first
FAR = 1 << 32
ODD = L.Tensor(FAKE + 8, 1 << 20, 1 << 20, 64, 1)


def _t(h=2, s=8, d=64, at=FAKE, b=2):
    return L.Tensor(at, h * s * d, s * d, d, 1)


def _rotary(**kw):
    r = L.Rotary(L.BF16, 2, 4, 2, 8, 64, 64, 0, 0, 1.0, FAKE, None, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _norm(**kw):
    n = L.Norm(L.BF16, 1e-6, FAKE, FAKE)
    for k, v in kw.items():
        setattr(n, k, v)
    return n


ROTARY_BAD = [(dict(dtype=7), -2), (dict(batch=0), -1), (dict(seqlen=0), -1), (dict(head_dim=96), -3), (dict(rotary_dim=63), -1),
              (dict(inverse=1), -1), (dict(inv_freq=None), -1), (dict(batch=1 << 20, seqlen=1 << 12), -4)]
NORM_BAD = [(dict(weight_dtype=L.F16), -2), (dict(weight_dtype=5), -2), (dict(eps=0.0), -1), (dict(eps=-1.0), -1),
            (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(eps=1e-40), -1), (dict(q_weight=None), -1),
            (dict(k_weight=None), -1), (dict(q_weight=FAKE + 1), -5), (dict(weight_dtype=L.F32, k_weight=FAKE + 2), -5)]


@pytest.mark.parametrize("r,n,code", [(r, {}, c) for r, c in ROTARY_BAD] + [({}, n, c) for n, c in NORM_BAD]
                         + [({}, None, -1), (dict(heads_kv=0), {}, -1)])
def test_norm_refuses(r, n, code):
    lib, r, n = L.load(), _rotary(**r), None if n is None else _norm(**n)
    q, k, cache = _t(4), _t(2), _t(2, 100, at=FAR)
    assert lib.flexatt_norm_rotary_apply(r, n, q, k, q, k, None) == code
    assert lib.flexatt_norm_rotary_grad(r, n, q, k, q, k, q, k, FAKE, FAKE, FAKE, 1 << 40, None) == code
    assert lib.flexatt_norm_rotary_append(r, n, q, k, k, q, cache, _t(2, 100, at=2 * FAR), 100, FAKE, None) == code
    if n is not None:
        assert lib.flexatt_quant_append(r, n, L.INT8, q, k, k, q, cache, _t(2, 100, at=2 * FAR), 3 * FAR, 4 * FAR, 100, FAKE,
                                        None) == code


def test_norm_refuses_tensors():
    lib, r, n, q, k = L.load(), _rotary(), _norm(), _t(4), _t(2)
    same = L.Tensor(FAKE, 0, 512, 64, 1)  # two sequences at one place: fine to read, not to write
    for args in ((ODD, k, q, k), (q, ODD, q, k), (q, k, same, k), (q, k, q, same)):
        assert lib.flexatt_norm_rotary_apply(r, n, *args, None) == -5
    call = lambda q=q, k=k, gq=q, gk=k, dq=q, dk=k, wq=FAKE, wk=FAKE, ws=FAKE, size=1 << 40, r=r: \
        lib.flexatt_norm_rotary_grad(r, n, q, k, gq, gk, dq, dk, wq, wk, ws, size, None)  # noqa: E731
    assert call(q=ODD) == call(k=ODD) == call(gq=ODD) == call(gk=ODD) == call(dq=same) == call(dk=same) == -5
    assert call(wq=None) == call(wk=None) == call(ws=None) == call(size=lib.flexatt_norm_rotary_grad_workspace(r) - 1) == -1
    assert call(ws=FAKE + 4) == call(wq=FAKE + 1) == call(wk=FAKE + 1) == -5
    assert lib.flexatt_norm_rotary_grad_workspace(_rotary(dtype=9)) == 2 ** 64 - 1
    alone = L.Norm(L.BF16, 1e-6, FAKE, None)
    for k_of in (dict(k=k), dict(k_out=k)):
        a = dict(dict(k=None, k_out=None), **k_of)
        assert lib.flexatt_norm_rotary_apply(_rotary(heads_kv=0), alone, q, a["k"], q, a["k_out"], None) == -1


@pytest.mark.parametrize("dtype,B,S,D,code", [
    (L.BF16, 1, 1 << 28, 256, -6), (L.BF16, 1, (1 << 28) - 16, 256, -5), (L.F32, 1, 1 << 27, 256, -6),
    (L.F16, 2, 1 << 28, 128, -6), (L.F16, 2, (1 << 28) - 64, 128, -5)])
def test_norm_launch_limits(dtype, B, S, D, code):
    r = L.Rotary(dtype, B, 1, 0, S, D, 0, 0, 0, 1.0, None, None, 0, 0, 0, 0)
    assert L.load().flexatt_norm_rotary_apply(r, L.Norm(dtype, 1e-6, FAKE, None), ODD, None, ODD, None, None) == code


def _append(**kw):
    a = dict(r=_rotary(), n=None, code=L.E4M3, q=_t(4), k=_t(), v=_t(), qo=_t(4), kc=_t(2, 100, at=FAR),
             vc=_t(2, 100, at=2 * FAR), ks=3 * FAR, vs=4 * FAR, rows=100, lengths=FAKE)
    a.update(kw)
    return L.load().flexatt_quant_append(*a.values(), None)


def test_quantized_append_refuses():
    assert _append(code=0) == _append(code=3) == _append(ks=None) == _append(vs=None) == _append(rows=0) == -1
    assert _append(lengths=None) == _append(r=_rotary(inverse=1)) == _append(r=_rotary(heads_kv=0)) == -1
    assert _append(rows=1 << 30) == -4
    assert _append(ks=3 * FAR + 2) == _append(vs=4 * FAR + 1) == -5
    assert _append(kc=L.Tensor(FAR, 12800, 6400, 72, 1)) == -5   # rows off 16-byte boundaries
    assert _append(vc=L.Tensor(FAR, 12800, 0, 64, 1)) == -5      # heads at one place
    assert _append(vc=_t(2, 100, at=FAR + 64)) == -5             # keys and values on each other
    big = 2 * 2 * 100 * 64
    for edge in (0, big - 16):
        for name, heads in (("q", 4), ("qo", 4), ("k", 2), ("v", 2)):
            for cache in (FAR, 2 * FAR, 3 * FAR, 4 * FAR):
                at = cache + (edge if cache <= 2 * FAR else edge and 2 * 2 * 100 * 4 - 16)
                assert _append(**{name: _t(heads, at=at)}) == -5, (name, cache, edge)
    assert _append(ks=FAR + 16) == _append(vs=2 * FAR + big - 4) == _append(ks=4 * FAR + 4) == _append(vs=3 * FAR - 4) == -5
    assert _append(lengths=FAR + 8) == _append(lengths=3 * FAR + 8) == -5


def _dequant(**kw):
    p = L.Dequant(L.BF16, L.INT8, 2, 2, 100, 64, 1, 0, FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=4), -2), (dict(code=0), -1), (dict(code=3), -1), (dict(batch=0), -1), (dict(cache_rows=0), -1),
    (dict(head_dim=48), -3), (dict(fill=2), -1), (dict(reserved=1), -1), (dict(lengths=None), -1),
    (dict(batch=1 << 16, cache_rows=1 << 16), -4), (dict(dtype=L.F32, head_dim=256, batch=1, cache_rows=1 << 27), -6)])
def test_dequant_refuses(kw, code):
    c, o, p = _t(2, 100), _t(2, 100, at=FAR), _t(2, 100, at=2 * FAR)
    assert L.load().flexatt_dequant_rows(_dequant(**kw), c, c, FAKE, FAKE, o, p, None) == code


def test_dequant_refuses_tensors():
    c, o, p = _t(2, 100), _t(2, 100, at=FAR), _t(2, 100, at=2 * FAR)
    call = lambda k=c, v=c, ks=FAKE, vs=FAKE, ko=o, vo=p, d=None: \
        L.load().flexatt_dequant_rows(d or _dequant(), k, v, ks, vs, ko, vo, None)  # noqa: E731
    assert call(k=ODD) == call(v=ODD) == call(ko=ODD) == call(vo=o) == call(ks=FAKE + 2) == call(vs=FAKE + 1) == -5
    assert call(ks=None) == call(vs=None) == -1
    size = 2 * 2 * 100 * 128
    for at in (FAR, FAR + size - 16, 2 * FAR):
        assert call(k=_t(2, 100, at=at)) == call(v=_t(2, 100, at=at)) == call(ks=at) == call(vs=at) == -5
        assert call(d=_dequant(lengths=at)) == -5


def _tree(**kw):
    p = L.Tree(L.BF16, 2, 4, 2, 8, 64, 64, 0.125, 0.0, 0, 0, 0, None, None, FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=L.F32), -2), (dict(dtype=9), -2), (dict(batch=0), -1), (dict(tokens=0), -1), (dict(head_dim=80), -3),
    (dict(heads_kv=3), -4), (dict(scale=float("nan")), -1), (dict(soft_cap=-1.0), -1), (dict(sliding_window=-1), -1),
    (dict(lengths=None), -1), (dict(mask_batch=1), -1), (dict(tree_mask=FAKE, mask_batch=2, sliding_window=5), -1),
    (dict(heads_q=2, tokens=(1 << 20) + 1), -6)])
def test_quant_tree_refuses(kw, code):
    lib = L.load()
    c = _t(2, 64)
    assert lib.flexatt_quant_tree_fwd(_tree(**kw), L.INT8, _t(4), c, c, FAKE, FAKE, _t(4), FAKE, FAKE, 1 << 40, None) == code
    assert lib.flexatt_quant_tree_fwd_workspace(_tree(**kw)) == 2 ** 64 - 1


def test_quant_tree_refuses_tensors_and_workspace():
    lib, p = L.load(), _tree(cache_rows=8192)
    n = lib.flexatt_quant_tree_fwd_workspace(p)
    assert 0 < n < 1 << 30
    q, c = _t(4), _t(2, 8192)
    call = lambda code=L.E4M3, q=q, k=c, v=c, ks=FAKE, vs=FAKE, o=q, lse=FAKE, ws=FAKE, size=n: \
        lib.flexatt_quant_tree_fwd(p, code, q, k, v, ks, vs, o, lse, ws, size, None)  # noqa: E731
    assert call(code=0) == call(code=4) == call(ks=None) == call(vs=None) == call(lse=None) == call(ws=None) == -1
    assert call(size=n - 1) == -1
    far = L.Tensor(FAKE, 1 << 40, 64, 1 << 26, 1)  # rows 2^26 bytes apart
    assert call(k=far) == call(v=far) == -6
    assert call(q=ODD) == call(k=ODD) == call(v=ODD) == call(ks=FAKE + 2) == call(vs=FAKE + 2) == call(ws=FAKE + 8) == -5
    assert call(o=L.Tensor(FAKE, 0, 512, 64, 1)) == -5


@pytest.mark.parametrize("kw,rows,code", [
    (dict(dtype=9), 50, -2), (dict(batch=0), 50, -1), (dict(tokens=0), 50, -1), (dict(head_dim=80), 50, -3),
    (dict(heads_kv=3), 50, -4), (dict(scale=float("nan")), 50, -1), (dict(soft_cap=-1.0), 50, -1),
    (dict(lengths=None), 50, -1), (dict(tree_mask=FAKE, mask_batch=2, sliding_window=5), 50, -1), ({}, 0, -1), ({}, -3, -1),
    ({}, 1 << 30, -4), (dict(heads_q=2, tokens=(1 << 20) + 1), 50, -6)])
def test_prefix_refuses(kw, rows, code):
    lib, c, pre = L.load(), _t(2, 64), _t(2, 50)
    assert lib.flexatt_prefix_fwd(_tree(**kw), rows, _t(4), pre, pre, c, c, _t(4), FAKE, FAKE, 1 << 40, None) == code
    assert lib.flexatt_prefix_fwd_workspace(_tree(**kw), rows) == 2 ** 64 - 1


def test_prefix_refuses_tensors_and_workspace():
    lib, p = L.load(), _tree(cache_rows=8192)
    n = lib.flexatt_prefix_fwd_workspace(p, 5000)
    assert 0 < n < 1 << 30
    q, c, pre = _t(4), _t(2, 8192), _t(2, 5000)
    call = lambda q=q, pk=pre, pv=pre, k=c, v=c, o=q, lse=FAKE, ws=FAKE, size=n: \
        lib.flexatt_prefix_fwd(p, 5000, q, pk, pv, k, v, o, lse, ws, size, None)  # noqa: E731
    assert call(pk=None) == call(pv=None) == call(lse=None) == call(ws=None) == call(size=n - 1) == -1
    far = L.Tensor(FAKE, 1 << 40, 64, 1 << 25, 1)  # rows 2^26 bytes apart
    assert call(pk=far) == call(pv=far) == call(k=far) == call(v=far) == -6
    assert call(q=ODD) == call(pk=ODD) == call(pv=ODD) == call(k=ODD) == call(v=ODD) == call(ws=FAKE + 8) == -5
    assert call(o=L.Tensor(FAKE, 0, 512, 64, 1)) == -5


def test_cpu_tensors_have_no_fallback():
    x, w, f = torch.randn(1, 2, 4, 64), torch.ones(64), rot.rotary_frequencies(64)[0]
    c, s, n = torch.zeros(1, 2, 8, 64, dtype=torch.int8), torch.zeros(1, 2, 8), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: rot.norm_rotary_embedding(x, x, w, w, f), lambda: fc.norm_rotary_append(x, x, x, x, x, n, w, w, f),
                 lambda: fc.quantized_append(x, x, x, c, c, s, s, n, f), lambda: fc.dequantize_cache(c, c, s, s, n),
                 lambda: fc.quantized_tree_attention(x, c, c, s, s, n),
                 lambda: fc.shared_prefix_attention(x, x[0], x[0], x, x, n)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()
    with pytest.raises(RuntimeError, match="out must be"):
        fc.dequantize_cache(c, c, s, s, n, out=(x, None))


@pytest.mark.parametrize("inter", [False, True])
def test_oracle_gradient_is_the_forwards(inter):
    """The oracle's gradients against torch's own of its forward, in 64 bits."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 5, 32, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(32, generator=g, dtype=torch.float64, requires_grad=True)
    f, m = rot.rotary_frequencies(24, scaling="yarn", factor=4.0, original_length=64)
    at = torch.randint(0, 999, (2, 5), generator=g)
    y, _ = orc.norm_rotary(x, w, f, at, inter, m, 1e-3)
    gy = torch.randn(y.shape, generator=g, dtype=torch.float64)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    (ox, _), (ow, _) = orc.norm_rotary_grad(x.detach(), w.detach(), gy, f, at, inter, m, 1e-3)
    assert torch.allclose(dx, ox, rtol=1e-12, atol=1e-13) and torch.allclose(dw, ow, rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("Hq,Hkv,S,apply,append", [
    (1, 1, 1 << 26, -6, -6), (1, 1, (1 << 26) - 8, -5, -6), (1, 1, 44739240, -5, -5), (1, 1, 44739248, -5, -6),
    (1 << 30, 1, 1, -6, -6), ((1 << 30) - 1, 1, 1, -5, -5)])
def test_norm_launch_limits_of_keys_and_values(Hq, Hkv, S, apply, append):
    """Eight tokens of 1 KB a workgroup, for q, k and v each: 2^24 of 256 threads are one too many."""
    lib, n = L.load(), L.Norm(L.F32, 1e-6, FAKE, FAKE)
    r = L.Rotary(L.F32, 1, Hq, Hkv, S, 256, 0, 0, 0, 1.0, None, None, 0, 0, 0, 0)
    assert lib.flexatt_norm_rotary_apply(r, n, ODD, ODD, ODD, ODD, None) == apply
    assert lib.flexatt_norm_rotary_append(r, n, ODD, ODD, ODD, ODD, ODD, ODD, 100, FAKE, None) == append
    assert lib.flexatt_quant_append(r, n, L.INT8, ODD, ODD, ODD, ODD, ODD, ODD, FAKE, FAKE, 100, FAKE, None) == append
    assert lib.flexatt_quant_append(r, None, L.INT8, ODD, ODD, ODD, ODD, ODD, ODD, FAKE, FAKE, 100, FAKE, None) == append


def test_what_an_append_reads_lies_apart_from_the_cache():
    lib, kc, vc = L.load(), _t(2, 100, at=FAR), _t(2, 100, at=2 * FAR)
    wide = 2 * 2 * 100 * 128  # bytes of a cache of 16 bits, half of it one of 8

    def both(r=None, n=None):
        r, n = _rotary(**(r or {})), _norm(**(n or {}))
        a = lib.flexatt_norm_rotary_append(r, n, _t(4), _t(), _t(), _t(4), kc, vc, 100, FAKE, None)
        return a, lib.flexatt_quant_append(r, n, L.INT8, _t(4), _t(), _t(), _t(4), kc, vc, 3 * FAR, 4 * FAR, 100, FAKE, None)

    for at in (FAR, 2 * FAR, FAR + wide // 2 - 8, 2 * FAR + wide // 2 - 8, FAR - 8):
        assert both(r=dict(inv_freq=at)) == both(n=dict(q_weight=at)) == both(n=dict(k_weight=at)) == (-5, -5)
        assert both(r=dict(positions=at, position_bytes=8, position_stride_s=1)) == (-5, -5)
    # positions whose sequences lie one behind the other, or backwards
    assert both(r=dict(positions=FAR - 64, position_bytes=8, position_stride_b=8, position_stride_s=1)) == (-5, -5)
    assert both(r=dict(positions=FAR + wide // 2, position_bytes=4, position_stride_b=0, position_stride_s=-1)) == (-5, -5)
    for at in (3 * FAR, 4 * FAR, 4 * FAR + 2 * 2 * 100 * 4 - 8):
        assert both(r=dict(inv_freq=at))[1] == both(n=dict(q_weight=at))[1] == both(n=dict(k_weight=at))[1] == -5


def test_norm_gradients_lie_apart():
    lib, r, n = L.load(), _rotary(inv_freq=20 * FAR), _norm(q_weight=21 * FAR, k_weight=22 * FAR)
    ok = dict(q=_t(4, at=FAR), k=_t(2, at=2 * FAR), gq=_t(4, at=3 * FAR), gk=_t(2, at=4 * FAR), dq=_t(4, at=5 * FAR),
              dk=_t(2, at=6 * FAR), wq=7 * FAR, wk=8 * FAR, ws=9 * FAR, size=1 << 30)
    call = lambda **kw: lib.flexatt_norm_rotary_grad(r, n, *dict(ok, **kw).values(), None)  # noqa: E731
    for name, heads in (("dq", 4), ("dk", 2)):
        for other in (1, 2, 3, 4, 5 if name == "dk" else 6, 7, 8, 9, 20, 21, 22):
            assert call(**{name: _t(heads, at=other * FAR)}) == -5, (name, other)
    for name in ("wq", "wk", "ws"):
        for other in (1, 2, 3, 4, 5, 6, 20, 21, 22):
            assert call(**{name: other * FAR}) == -5, (name, other)
    assert call(wk=7 * FAR) == call(ws=7 * FAR) == call(ws=8 * FAR - 16) == -5


def test_mask_and_read_back_limits():
    lib, p = L.load(), _tree(batch=1, heads_q=1, heads_kv=1, tokens=1 << 15, cache_rows=1 << 16, tree_mask=FAKE, mask_batch=1)
    run = lambda: lib.flexatt_quant_tree_fwd(p, L.INT8, ODD, ODD, ODD, FAKE, FAKE, ODD, FAKE, FAKE, 1 << 40, None)  # noqa: E731
    assert run() == -5
    p.tokens += 1
    assert run() == -6 and lib.flexatt_quant_tree_fwd_workspace(p) == 2 ** 64 - 1
    p.tree_mask, p.mask_batch = None, 0
    assert run() == -5
    for rows, code in ((1 << 27, -6), ((1 << 27) - 16, -5)):  # 16 rows of 1 KB a workgroup
        d = _dequant(dtype=L.F32, head_dim=256, batch=1, cache_rows=rows)
        assert lib.flexatt_dequant_rows(d, ODD, ODD, FAKE, FAKE, ODD, ODD, None) == code
