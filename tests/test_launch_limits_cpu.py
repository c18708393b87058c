"""Calls of more work-items than one launch can have (2^32 - 1) are refused by the C entries; one less goes on to the next
check, a tensor off its 16-byte boundary.  No kernel is launched here."""
import pytest

import flexatt_lib as L

FAKE = 1 << 20  # never dereferenced
ODD = L.Tensor(FAKE + 8, 1 << 20, 1 << 20, 64, 1)


@pytest.mark.parametrize("dtype,B,S,D,rotary,code", [
    (L.BF16, 1, 1 << 28, 32, 10, -6), (L.BF16, 1, (1 << 28) - 16, 32, 10, -5),   # a thread per pair
    (L.F32, 4, 1 << 25, 64, 2, -6), (L.F32, 4, (1 << 25) - 8, 64, 2, -5),
    (L.BF16, 1, 1 << 28, 32, 16, -5), (L.F16, 2, 1 << 28, 128, 64, -6), (L.F16, 2, 1 << 27, 128, 64, -5),  # per 32 bytes
    (L.F32, 1, 1 << 27, 256, 256, -6), (L.F32, 1, (1 << 27) - 8, 256, 256, -5)])
def test_rotation(dtype, B, S, D, rotary, code):
    r = L.Rotary(dtype, B, 1, 0, S, D, rotary, 0, 0, 1.0, FAKE, None, 0, 0, 0, 0)
    assert L.load().flexatt_rotary_apply(r, ODD, None, ODD, None, None) == code
    r.heads_kv = 1
    assert L.load().flexatt_rotary_append(r, ODD, ODD, ODD, ODD, ODD, ODD, 1, FAKE, None) == code


@pytest.mark.parametrize("dtype,D,B,Hkv,Skv,code", [
    (L.BF16, 64, 1 << 20, 16, 1, -6), (L.BF16, 64, 1 << 20, 15, 100, -5), (L.BF16, 64, 1 << 19, 15, 256, -5),
    (L.F32, 256, 1 << 20, 8, 200, -6), (L.F32, 256, 1 << 20, 7, 200, -5)])
def test_weight_sums(dtype, D, B, Hkv, Skv, code):
    p = L.Weights(dtype, B, Hkv, Hkv, 1, Skv, D, 0.125, 0.0, 0, 0, 0, 0, 0, None, None)
    assert L.load().flexatt_weight_sums(p, ODD, ODD, FAKE, FAKE, None, 0, None) == code
    assert (L.load().flexatt_weight_sums_workspace(p) == 2 ** 64 - 1) == (code == -6)


@pytest.mark.parametrize("B,H,code", [(1 << 22, 4, -6), ((1 << 22) - 1, 4, -5)])
def test_eviction(B, H, code):
    e = L.Evict(L.BF16, B, H, 100, 64, 50, 0, 0, 50, 0, FAKE)
    assert L.load().flexatt_evict_rows(e, ODD, ODD, FAKE, ODD, ODD, FAKE, FAKE, FAKE, None) == code
