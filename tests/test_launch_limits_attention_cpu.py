"""Attention over a cache of 8 bits and behind a prefix: calls of more work-items than one launch can have (2^32 - 1) are
refused by the C entries and their workspace queries; the largest that fit go on to the next check, a tensor off its 16-byte
boundary.  No kernel is launched here.  (Without a GPU the plan is that of 256 CUs.)"""
import pytest

import flexatt_lib as L

FAKE = 1 << 20  # never dereferenced
ODD = L.Tensor(FAKE + 8, 1 << 20, 1 << 20, 64, 1)
NONE = 2 ** 64 - 1


def tree(dtype, B, Hq, Hkv, T, C, D):
    return L.Tree(dtype, B, Hq, Hkv, T, C, D, 0.125, 0.0, 0, 0, 0, None, None, FAKE)


@pytest.mark.parametrize("D,B,Hq,Hkv,T,C,code", [
    (128, 1 << 15, 256, 256, 1, 1, -6), (128, 1, 8388600, 8388600, 1, 1, -5), (128, 1, 8388601, 8388601, 1, 1, -6),
    (64, 1 << 15, 256, 256, 1, 1, -5), (256, 1 << 15, 256, 256, 1, 1, -5),  # 256 threads a workgroup, 512 above
    (128, 8388352, 1, 1, 1, 200, -5), (128, 8388601, 1, 1, 1, 200, -6),     # a cache this short is one chunk
    (128, 1 << 13, 1024, 32, 1, 100, -5), (128, 1 << 18, 32, 1, 1, 100, -5)])
def test_cache_of_8_bits(D, B, Hq, Hkv, T, C, code):
    lib = L.load()
    for dtype in (L.F16, L.BF16):
        p = tree(dtype, B, Hq, Hkv, T, C, D)
        assert lib.flexatt_quant_tree_fwd(p, L.INT8, ODD, ODD, ODD, FAKE, FAKE, ODD, FAKE, FAKE, 1 << 62, None) == code
        assert (lib.flexatt_quant_tree_fwd_workspace(p) == NONE) == (code == -6)


@pytest.mark.parametrize("dtype,D,B,Hkv,code", [
    (L.BF16, 128, 32639, 256, -5), (L.BF16, 128, 32640, 256, -6), (L.F16, 128, 1 << 15, 256, -6),  # eight row tiles each
    (L.BF16, 64, 32262, 256, -5), (L.BF16, 64, 32263, 256, -6), (L.F16, 32, 1 << 15, 256, -6),     # waves that share tiles
    (L.BF16, 256, 1 << 15, 256, -5), (L.F32, 256, 1 << 15, 256, -5), (L.F32, 64, 1 << 15, 256, -5)])
def test_prefix(dtype, D, B, Hkv, code):
    lib, p = L.load(), tree(dtype, B, Hkv, Hkv, 1, 1, D)
    assert lib.flexatt_prefix_fwd(p, 1, ODD, ODD, ODD, ODD, ODD, ODD, FAKE, FAKE, 1 << 62, None) == code
    assert (lib.flexatt_prefix_fwd_workspace(p, 1) == NONE) == (code == -6)
