"""Gradients of the norm: numbers of heads beyond 2^30, which the forward refuses, on the host.  No kernel is launched here."""
import pytest

import flexatt_lib as L

FAKE = 1 << 20  # never dereferenced
ODD = L.Tensor(FAKE + 8, 1 << 20, 1 << 20, 64, 1)
NONE = 2 ** 64 - 1


@pytest.mark.parametrize("Hq,Hkv,code", [(2 ** 31 - 1, 0, -6), (2 ** 31 - 1, 2 ** 31 - 1, -6), ((1 << 30) + 1, 0, -6),
                                         (1 << 30, 1, -6), (1 << 30, 0, -5), ((1 << 30) - 1, 1, -5), (1, (1 << 30) - 1, -5)])
def test_gradients_of_many_heads(Hq, Hkv, code):
    lib, n = L.load(), L.Norm(L.BF16, 1e-6, FAKE, FAKE if Hkv else None)
    r = L.Rotary(L.BF16, 1, Hq, Hkv, 1, 32, 0, 0, 0, 1.0, None, None, 0, 0, 0, 0)
    k, dk = (ODD, FAKE) if Hkv else (None, None)
    assert lib.flexatt_norm_rotary_grad(r, n, ODD, k, ODD, k, ODD, k, FAKE, dk, FAKE, 1 << 40, None) == code
    assert lib.flexatt_norm_rotary_apply(r, n, ODD, k, ODD, k, None) == code
    size = lib.flexatt_norm_rotary_grad_workspace(r)
    assert size == NONE if code == -6 else 0 < size <= 4096 * 32 * 4
