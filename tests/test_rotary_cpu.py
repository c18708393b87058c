"""Rotary positions on the host: frequencies and their scalings, and the refusals of both entry points' arguments.
No kernel is launched here."""
import math

import pytest
import torch

import flexatt_lib as L
import flexatt_rotary as rot

FAKE = 1 << 20  # aligned, never dereferenced: every call below fails its checks first


def test_frequencies_without_scaling():
    f, m = rot.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], dtype=torch.float64), rtol=1e-15)


def test_linear_and_ntk_scaling():
    f0, _ = rot.rotary_frequencies(64)
    f1, m1 = rot.rotary_frequencies(64, scaling="linear", factor=4.0)
    f2, m2 = rot.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert m1 == m2 == 1.0
    assert torch.allclose(f1, f0 / 4, rtol=1e-15)
    assert f2[0] == f0[0] and torch.allclose(f2[-1], f0[-1] / 4, rtol=1e-12)  # fastest kept, slowest divided


@pytest.mark.parametrize("scaling", ["turns", "yarn"])
def test_blended_scalings(scaling):
    kw = dict(base=500000.0, factor=8.0, original_length=8192, fast=4.0 if scaling == "turns" else 32.0)
    f0, _ = rot.rotary_frequencies(128, base=500000.0)
    f, m = rot.rotary_frequencies(128, scaling=scaling, **kw)
    turns = 8192 * f0 / (2 * math.pi)
    assert torch.equal(f[turns > 64], f0[turns > 64])            # fast pairs stay
    assert torch.allclose(f[turns < 0.5], f0[turns < 0.5] / 8, rtol=1e-15)  # slow ones are interpolated
    assert bool((f <= f0).all()) and bool((f >= f0 / 8 * (1 - 1e-15)).all()) and bool((f[1:] <= f[:-1]).all())
    assert m == (1.0 if scaling == "turns" else pytest.approx(0.1 * math.log(8.0) + 1.0))


def test_turns_scaling_is_linear_between():
    f0, _ = rot.rotary_frequencies(128, base=500000.0)
    f, _ = rot.rotary_frequencies(128, base=500000.0, scaling="turns", factor=8.0, original_length=8192, fast=4.0)
    turns = 8192 * f0 / (2 * math.pi)
    mid = (turns > 1) & (turns < 4)
    assert bool(mid.any())
    share = (turns[mid] - 1) / 3
    assert torch.allclose(f[mid], f0[mid] * share + f0[mid] / 8 * (1 - share), rtol=1e-14)


@pytest.mark.parametrize("args,kw", [
    ((7,), {}), ((0,), {}), ((8,), dict(scaling="other")), ((8,), dict(scaling="linear", factor=0.5)),
    ((8,), dict(scaling="turns", factor=2.0)), ((8,), dict(scaling="yarn", factor=2.0, original_length=10, fast=1.0)),
    ((2,), dict(scaling="ntk", factor=2.0))])
def test_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        rot.rotary_frequencies(*args, **kw)


def test_cpu_tensors_have_no_fallback():
    q = torch.randn(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        rot.rotary_embedding(q, q, rot.rotary_frequencies(64)[0])


def _rotary(**kw):
    r = L.Rotary(L.BF16, 2, 4, 2, 8, 64, 64, 0, 0, 1.0, FAKE, None, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _t(h, s=8, d=64):
    return L.Tensor(FAKE, h * s * d, s * d, d, 1)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), -2), (dict(batch=0), -1), (dict(heads_q=0), -1), (dict(seqlen=0), -1), (dict(head_dim=96), -3),
    (dict(heads_kv=-1), -1), (dict(rotary_dim=63), -1), (dict(rotary_dim=66), -1), (dict(rotary_dim=-2), -1),
    (dict(inv_freq=None), -1), (dict(inv_freq=FAKE + 4), -5), (dict(interleaved=2), -1), (dict(inverse=2), -1),
    (dict(magnitude=float("inf")), -1), (dict(reserved=1), -1), (dict(positions=FAKE), -1),
    (dict(positions=FAKE, position_bytes=2), -1), (dict(positions=FAKE + 4, position_bytes=8), -5),
    (dict(position_bytes=4), -1), (dict(batch=1 << 20, seqlen=1 << 12), -4)])
def test_capi_refuses(kw, code):
    lib = L.load()
    assert lib.flexatt_rotary_apply(_rotary(**kw), _t(4), _t(2), _t(4), _t(2), None) == code


def test_capi_refuses_tensors():
    lib = L.load()
    r, q, k = _rotary(), _t(4), _t(2)
    odd = L.Tensor(FAKE + 8, 2048, 512, 64, 1)
    bad = L.Tensor(FAKE, 0, 512, 64, 1)  # two sequences at one place: fine to read, not to write
    assert lib.flexatt_rotary_apply(r, odd, k, q, k, None) == -5
    assert lib.flexatt_rotary_apply(r, q, odd, q, k, None) == -5
    assert lib.flexatt_rotary_apply(r, q, k, bad, k, None) == -5
    assert lib.flexatt_rotary_apply(r, q, k, q, bad, None) == -5
    assert lib.flexatt_rotary_apply(r, q, None, q, None, None) == -1
    assert lib.flexatt_rotary_apply(_rotary(heads_kv=0), q, k, q, k, None) == -1


def test_capi_append_refuses():
    lib = L.load()
    q, k = _t(4), _t(2)
    far = 1 << 30
    cache = L.Tensor(far, 2 * 100 * 64, 100 * 64, 64, 1)
    call = lambda r=None, q=q, k=k, v=k, qo=q, kc=cache, vc=cache, rows=100, n=FAKE: lib.flexatt_rotary_append(  # noqa: E731
        r or _rotary(), q, k, v, qo, kc, vc, rows, n, None)
    assert call(r=_rotary(heads_kv=0)) == -1
    assert call(rows=0) == -1 and call(n=None) == -1
    assert call(rows=1 << 30) == -4
    assert call(kc=L.Tensor(far, 2 * 100 * 64, 100 * 64, 60, 1)) == -5   # rows not on 16-byte boundaries
    assert call(vc=L.Tensor(far, 2 * 100 * 64, 0, 64, 1)) == -5          # heads at one place
    assert call(k=L.Tensor(far + 64, 1024, 512, 64, 1)) == -5            # the tokens overlap the cache
    assert call(v=L.Tensor(far + 64, 1024, 512, 64, 1)) == -5
    assert call() == -5                                                  # one cache for keys and values
