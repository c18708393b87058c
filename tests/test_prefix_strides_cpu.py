"""A prefix [Hkv, P, D] has no batch: the C entry takes its tensors whatever their batch stride is.  No kernel is launched."""
import pytest

import flexatt_lib as L

FAKE = 1 << 20  # never dereferenced


def _t(rows, heads=2, d=64, **kw):
    t = L.Tensor(FAKE, heads * rows * d, rows * d, d, 1)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("stride", [-64, 3, 0, 1 << 62])
def test_batch_stride_is_not_used(stride):
    p = L.Tree(L.BF16, 2, 4, 2, 8, 64, 64, 0.125, 0.0, 0, 0, 0, None, None, FAKE)
    q, c, pre, odd = _t(8, 4), _t(64), _t(50), _t(50, stride_b=stride)
    call = lambda pk, pv: \
        L.load().flexatt_prefix_fwd(p, 50, q, pk, pv, c, c, q, None, FAKE, 1 << 40, None)  # noqa: E731
    assert call(odd, pre) == call(pre, odd) == call(pre, pre) == -1  # all but the LSE, which is missing
    assert call(_t(50, stride_h=3), pre) == call(pre, _t(50, stride_s=-64)) == -5
    assert call(None, pre) == call(pre, None) == -1
