"""Outputs of the cache calls that lie on an input or on each other are refused by the C entries, before any launch."""
import pytest

import flexatt_lib as L


def tensor(at, heads, rows, D=64, B=2):
    return L.Tensor(at, heads * rows * D, rows * D, D, 1)  # aligned, never dereferenced


@pytest.mark.parametrize("which", ["q", "k", "lse", "starts", "lengths", None])
@pytest.mark.parametrize("end", ["first", "last"])
def test_weight_sums_lie_apart_from_their_inputs(which, end):
    """Many query rows over few keys, which takes a workspace: leaving it out is what a call without overlaps fails with."""
    at = dict(q=1 << 24, k=1 << 25, lse=1 << 26, starts=1 << 27, lengths=1 << 28)
    size = dict(q=2 * 4 * 4096 * 128, k=2 * 2 * 64 * 128, lse=2 * 4 * 4096 * 4, starts=8, lengths=8)
    p = L.Weights(L.BF16, 2, 4, 2, 4096, 64, 64, 0.125, 0.0, 0, 0, 0, 1, 0, at["starts"], at["lengths"])
    assert L.load().flexatt_weight_sums_workspace(p) > 0
    sums, bytes_ = 1 << 29, 2 * 2 * 64 * 4
    if which:
        sums = at[which] - bytes_ + 4 if end == "first" else at[which] + size[which] - 4
    code = L.load().flexatt_weight_sums(p, tensor(at["q"], 4, 4096), tensor(at["k"], 2, 64), at["lse"], sums, None, 0, None)
    assert code == (-5 if which else -1)


@pytest.mark.parametrize("which", ["q", "q_out", "k", "v", "lengths"])
@pytest.mark.parametrize("cache", ["k_cache", "v_cache"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_appended_tokens_lie_apart_from_the_cache(which, cache, end):
    at = dict(q=1 << 24, q_out=1 << 25, k=1 << 26, v=1 << 27, lengths=1 << 28, k_cache=1 << 30, v_cache=1 << 31)
    size = dict(q=2 * 4 * 8 * 128, q_out=2 * 4 * 8 * 128, k=2 * 2 * 8 * 128, v=2 * 2 * 8 * 128, lengths=8)
    at[which] = at[cache] - size[which] + 16 if end == "first" else at[cache] + 2 * 2 * 100 * 128 - 16
    if which == "lengths" and end == "first":
        at[which] = at[cache] - 4
    r = L.Rotary(L.BF16, 2, 4, 2, 8, 64, 0, 0, 0, 1.0, None, None, 0, 0, 0, 0)
    heads = dict(q=4, q_out=4, k=2, v=2)
    t = {n: tensor(at[n], heads[n], 8) for n in heads}
    c = [tensor(at[n], 2, 100) for n in ("k_cache", "v_cache")]
    assert L.load().flexatt_rotary_append(r, t["q"], t["k"], t["v"], t["q_out"], *c, 100, at["lengths"], None) == -5
