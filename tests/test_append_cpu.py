"""What the append's C entry takes and refuses.  No kernel is launched here: every call fails its last check."""
import pytest

import flexatt_lib as L

FAKE, FAR = 1 << 20, 1 << 30  # aligned, never dereferenced


def rotary(**kw):
    r = L.Rotary(L.BF16, 2, 4, 2, 8, 64, 64, 0, 0, 1.0, FAKE, None, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def tokens(heads, at=FAKE):
    return L.Tensor(at, heads * 8 * 64, 8 * 64, 64, 1)


def cache(at=FAR):
    return L.Tensor(at, 2 * 100 * 64, 100 * 64, 64, 1)


def append(r, q, qo, k=None, v=None, kc=None, vc=None):
    return L.load().flexatt_rotary_append(r, q, k or tokens(2), v or tokens(2), qo, kc or cache(), vc or cache(1 << 34),
                                          100, FAKE, None)


@pytest.mark.parametrize("kw,q,qo,code", [
    # keys and values alone: past every check of the query, to that of the last cache
    (dict(heads_q=0), None, None, -5), (dict(heads_q=0), tokens(4), tokens(4), -1), (dict(heads_q=0), None, tokens(4), -1),
    (dict(heads_q=0, heads_kv=0), None, None, -1), (dict(heads_q=-1), None, None, -1), (dict(), None, None, -1),
    (dict(heads_q=0, dtype=9), None, None, -2), (dict(heads_q=0, head_dim=80), None, None, -3)])
def test_append_without_query_heads(kw, q, qo, code):
    assert append(rotary(**kw), q, qo, vc=L.Tensor(1 << 34, 12800, 0, 64, 1)) == code
