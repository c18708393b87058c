"""The cache operators' refusals (Python and C ABI), their workspaces and their oracle, on the host.  No kernel is
launched here."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_lib as L
from oracle import cache_oracle as orc

FAKE = 1 << 20  # aligned, never dereferenced: every call below fails its checks first
CPU = torch.device("cpu")


def _t(h=2, s=64, d=64, at=FAKE):
    return L.Tensor(at, h * s * d, s * d, d, 1)


def _tree(**kw):
    p = L.Tree(L.BF16, 2, 4, 2, 8, 64, 64, 0.125, 0.0, 0, 0, 0, None, None, FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


TREE_BAD = [
    (dict(dtype=9), -2), (dict(batch=0), -1), (dict(tokens=0), -1), (dict(cache_rows=0), -1), (dict(head_dim=80), -3),
    (dict(heads_kv=3), -4), (dict(heads_kv=0), -1), (dict(scale=float("nan")), -1), (dict(soft_cap=-1.0), -1),
    (dict(soft_cap=float("inf")), -1), (dict(sliding_window=-1), -1), (dict(reserved=1), -1), (dict(lengths=None), -1),
    (dict(mask_batch=1), -1), (dict(tree_mask=FAKE), -1), (dict(tree_mask=FAKE, mask_batch=3), -1),
    (dict(tree_mask=FAKE, mask_batch=2, sliding_window=5), -1), (dict(batch=1 << 16, cache_rows=1 << 16), -4),
    (dict(batch=1, heads_kv=1, heads_q=1, cache_rows=(1 << 30) + 1), -4),
    (dict(heads_q=2, tokens=(1 << 20) + 1), -6), (dict(batch=1 << 12, heads_q=2, tokens=1 << 11), -6)]


@pytest.mark.parametrize("kw,code", TREE_BAD)
def test_tree_capi_refuses(kw, code):
    lib = L.load()
    assert lib.flexatt_tree_fwd(_tree(**kw), _t(4, 8), _t(), _t(), _t(4, 8), FAKE, FAKE, 1 << 40, None) == code
    assert lib.flexatt_tree_fwd_workspace(_tree(**kw)) == 2 ** 64 - 1


def test_tree_capi_refuses_tensors_and_workspace():
    lib = L.load()
    p = _tree(cache_rows=8192)
    n = lib.flexatt_tree_fwd_workspace(p)
    assert 0 < n < 1 << 30
    q, c = _t(4, 8), _t(2, 8192)
    odd = L.Tensor(FAKE + 8, 2048, 512, 64, 1)
    assert lib.flexatt_tree_fwd(p, odd, c, c, q, FAKE, FAKE, n, None) == -5
    assert lib.flexatt_tree_fwd(p, q, odd, c, q, FAKE, FAKE, n, None) == -5
    assert lib.flexatt_tree_fwd(p, q, c, odd, q, FAKE, FAKE, n, None) == -5
    assert lib.flexatt_tree_fwd(p, q, c, c, L.Tensor(FAKE, 0, 512, 64, 1), FAKE, FAKE, n, None) == -5
    # rows 2^26 bytes apart: their offsets within a tile would leave 32 bits
    far = L.Tensor(FAKE, 1 << 40, 64, 1 << 25, 1)
    assert lib.flexatt_tree_fwd(p, q, far, c, q, FAKE, FAKE, n, None) == -6
    assert lib.flexatt_tree_fwd(p, q, c, far, q, FAKE, FAKE, n, None) == -6
    assert lib.flexatt_tree_fwd(p, q, c, c, q, None, FAKE, n, None) == -1
    assert lib.flexatt_tree_fwd(p, q, c, c, q, FAKE, None, 0, None) == -1
    assert lib.flexatt_tree_fwd(p, q, c, c, q, FAKE, FAKE, n - 1, None) == -1
    assert lib.flexatt_tree_fwd(p, q, c, c, q, FAKE, FAKE + 4, n, None) == -5


def _weights(**kw):
    p = L.Weights(L.BF16, 2, 4, 2, 8, 64, 64, 0.125, 0.0, 1, 0, 0, 0, 0, None, None)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=-1), -2), (dict(seqlen_q=0), -1), (dict(seqlen_kv=0), -1), (dict(head_dim=48), -3),
    (dict(heads_kv=3), -4), (dict(scale=float("inf")), -1), (dict(soft_cap=float("nan")), -1), (dict(causal=2), -1),
    (dict(accumulate=3), -1), (dict(sliding_window=-4), -1), (dict(reserved=9), -1),
    (dict(batch=1, heads_q=2, heads_kv=1, seqlen_q=(1 << 29) + 1), -4)])
def test_weights_capi_refuses(kw, code):
    lib = L.load()
    assert lib.flexatt_weight_sums(_weights(**kw), _t(4, 8), _t(), FAKE, FAKE, FAKE, 1 << 40, None) == code
    assert lib.flexatt_weight_sums_workspace(_weights(**kw)) == 2 ** 64 - 1


def test_weights_capi_refuses_tensors():
    lib = L.load()
    odd = L.Tensor(FAKE, 2048, 512, 60, 1)
    assert lib.flexatt_weight_sums(_weights(), odd, _t(), FAKE, FAKE, FAKE, 1 << 40, None) == -5
    assert lib.flexatt_weight_sums(_weights(), _t(4, 8), odd, FAKE, FAKE, FAKE, 1 << 40, None) == -5
    assert lib.flexatt_weight_sums(_weights(), _t(4, 8), _t(), None, FAKE, FAKE, 1 << 40, None) == -1
    assert lib.flexatt_weight_sums(_weights(), _t(4, 8), _t(), FAKE, None, FAKE, 1 << 40, None) == -1


def _evict(**kw):
    p = L.Evict(L.BF16, 2, 2, 64, 64, 32, 8, 4, 32, 0, FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -2), (dict(cache_rows=0), -1), (dict(head_dim=100), -3), (dict(keep=0), -1), (dict(recent=-1), -1),
    (dict(sinks=-1), -1), (dict(recent=20, sinks=13), -1), (dict(out_rows=31), -1), (dict(fill=2), -1),
    (dict(lengths=None), -1), (dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1), -1)])
def test_evict_capi_refuses(kw, code):
    lib = L.load()
    far = 1 << 30
    out = _t(2, 32, 64, far)
    assert lib.flexatt_evict_rows(_evict(**kw), _t(), _t(), FAKE, out, out, far, far, far, None) == code


def test_evict_capi_refuses_overlap():
    lib = L.load()
    far = 1 << 30
    out, c = _t(2, 32, 64, far), _t()
    args = [_evict(), c, c, FAKE, out, out, far, far, far, None]
    for i, inside in ((4, _t(2, 32, 64, FAKE + 128)), (5, c), (6, FAKE + 64), (7, FAKE), (8, FAKE)):
        bad = list(args)
        bad[i] = inside
        assert lib.flexatt_evict_rows(*bad) == -5
    assert lib.flexatt_evict_rows(*args) == -5  # k_out is v_out
    for i in (1, 2, 3, 4, 5, 6, 7, 8):
        bad = list(args)
        bad[i] = None
        assert lib.flexatt_evict_rows(*bad) == -1


# ------------------------------------------------------------------------ Python --
def test_cpu_tensors_have_no_fallback():
    q, c, n = torch.randn(1, 2, 4, 64), torch.randn(1, 2, 32, 64), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fc.tree_attention(q, c, c, n)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fc.rotary_append(q, q, q, c, c, n, None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fc.attention_weight_sums(q, c, torch.zeros(1, 2, 4))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fc.evict_cache(c, c, torch.zeros(1, 2, 32), n, 8)
    for f in (lambda: fc.tree_attention(None, c, c, n), lambda: fc.attention_weight_sums([1], c, None),
              lambda: fc.evict_cache(None, c, None, n, 8), lambda: fc.rotary_append(1, q, q, c, c, n, None)):
        with pytest.raises(RuntimeError, match="torch.Tensor"):
            f()


def test_native_module_counts_its_arguments():
    c = L.native()
    assert c.ABI_VERSION == L.ABI_VERSION
    for f in (c.rotary, c.rotary_append, c.tree_attention, c.weight_sums, c.evict):
        with pytest.raises(TypeError):
            f()


def test_oracles_agree_with_plain_attention():
    """The tree oracle with a chain is causal attention at the end of the sequence; the weight oracle's sums over all
    keys are the number of rows."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 2, s, 32, generator=g, dtype=torch.float64) for s in (5, 20, 20))
    o, lse, _, _ = orc.tree_attention(q, k, v, [15])
    x = q @ k.transpose(2, 3) / 32 ** 0.5
    x = x.masked_fill(torch.arange(20) > torch.arange(15, 20)[:, None], float("-inf"))
    assert torch.allclose(o, torch.softmax(x, -1) @ v) and torch.allclose(lse, torch.logsumexp(x, -1))
    w, _ = orc.weight_sums(q, k, lse, causal=True, starts=15)
    assert torch.allclose(w.sum(-1), torch.full((1, 2), 5.0, dtype=torch.float64))


def test_oracle_eviction_order():
    nan, inf = float("nan"), float("inf")
    s = [5.0, 1.0, nan, 1.0, inf, 0.0, -0.0, 2.0]
    assert orc.evict(s, 8, 3, 0, 0) == [0, 2, 4]
    assert orc.evict(s, 8, 3, 1, 0) == [2, 4, 7]
    assert orc.evict(s, 8, 5, 0, 2) == [0, 1, 2, 4, 7]
    assert orc.evict(s, 8, 6, 0, 0) == [0, 1, 2, 3, 4, 7]
    assert orc.evict(s, 8, 7, 0, 0) == [0, 1, 2, 3, 4, 5, 7]  # of equal ones the first
    assert orc.evict(s, 3, 4, 0, 0) == [0, 1, 2]
