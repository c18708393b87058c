"""The workspace of tree attention: fp32 partials of the chunks that the kernel can cut, and no more.  (Without a GPU the
plan is that of 256 CUs.)"""
import itertools

import pytest

import flexatt_lib as L

FAKE = 1 << 20


def workspace(dtype, B, Hq, Hkv, T, C, D):
    return L.load().flexatt_tree_fwd_workspace(L.Tree(dtype, B, Hq, Hkv, T, C, D, 0.125, 0.0, 0, 0, 0, None, None, FAKE))


def plan(dtype, B, Hq, Hkv, T, C, D):
    """(workgroups at once for one group of row tiles, the least tiles of a chunk), as the launcher has them."""
    es = 4 if dtype == L.F32 else 2
    rows = -(-(Hq // Hkv) * T // 32)
    share = 1
    if es == 2 and D * es <= 256 and rows > 1:
        share = 4 if D * es > 128 and -(-rows // 4) * 24 <= -(-rows // 2) * 14 else 2
    groups = -(-rows // share)
    fit = 256 if D * es >= 256 else 512
    slots = fit // 8 // groups * 8 if groups <= fit // 8 else fit // groups
    return max(slots, 1), 16 if es == 2 and -(-C // 32) <= 16 else 8


def most_chunks(slots, least, Hkv, lengths):
    """Of one sequence, as the device cuts them: chunks longer than all tiles * Hkv / slots."""
    tiles = [-(-n // 32) for n in lengths]
    length = max(sum(tiles) * Hkv // slots + 1, least)
    return max(-(-t // length) for t in tiles)


@pytest.mark.parametrize("args", [(L.BF16, 4, 32, 8, 2048, 32768, 128), (L.F16, 2, 64, 64, 512, 9000, 64),
                                  (L.F32, 2, 32, 32, 300, 5000, 256), (L.BF16, 1, 8, 8, 8000, 100000, 128),
                                  (L.BF16, 64, 512, 512, 1, 4000, 32)])
def test_nothing_is_kept_where_no_sequence_can_be_cut(args):
    slots, _ = plan(*args)
    assert slots <= args[3]
    assert workspace(*args) == 0


@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
@pytest.mark.parametrize("Hkv,T,D", [(8, 1, 128), (8, 64, 64), (2, 53, 128), (1, 8, 256), (32, 300, 32)])
def test_partials_for_the_chunks_that_can_be(dtype, Hkv, T, D):
    """Room for every chunk that unequal lengths can make of one sequence, up to the launcher's own bound of twice the even
    share (three where shares are small), and for none that they cannot make."""
    G, C = 4, 40000
    for B in (1, 2, 7, 40):
        slots, least = plan(dtype, B, G * Hkv, Hkv, T, C, D)
        n = workspace(dtype, B, G * Hkv, Hkv, T, C, D)
        splits, rest = divmod(n - 4 * B * Hkv if n else 0, B * G * Hkv * T * (D + 1) * 4)
        splits = splits or 1
        assert rest == 0
        bound = 3 if 2 * B * Hkv > slots and B > 1 else 2 * -(-slots // (B * Hkv)) + 1
        can = max(most_chunks(slots, least, Hkv, (long,) + (short,) * (B - 1))
                  for long, short in itertools.product((C, C // 2, 3000), (C, 5000, T)))
        assert min(can, bound) <= splits <= max(-(-slots // Hkv), 1)
