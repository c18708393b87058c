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


PAIRS = [
    # offset of the second tensor in bytes, its strides over the first one's: memory in common
    (64, (1, 1, 1)), (128, (1, 1, 1)), (16, (1, 1, 1)), (100 * 128 - 128, (1, 1, 1)), (100 * 128, (1, 1, 1)),
    (2 * 2 * 100 * 128 - 16, (1, 1, 1)), (256, (1, 1, 2)), (3 * 100 * 128, (2, 1, 1)),
]


@pytest.mark.parametrize("offset,times", PAIRS)
@pytest.mark.parametrize("turn", [False, True])
def test_keys_and_values_share_no_memory(offset, times, turn):
    """Two tensors of 2 x 2 x 100 rows of 128 bytes that lie partly on each other, as the append's cache and as eviction's."""
    a = tensor(1 << 30, 2, 100)
    b = L.Tensor((1 << 30) + offset, 2 * 6400 * times[0], 6400 * times[1], 64 * times[2], 1)
    kc, vc = (b, a) if turn else (a, b)
    r = L.Rotary(L.BF16, 2, 4, 2, 8, 64, 0, 0, 0, 1.0, None, None, 0, 0, 0, 0)
    q, k = tensor(1 << 24, 4, 8), tensor(1 << 25, 2, 8)
    assert L.load().flexatt_rotary_append(r, q, k, k, q, kc, vc, 100, 1 << 26, None) == -5
    e = L.Evict(L.BF16, 2, 2, 300, 64, 100, 8, 4, 100, 0, 1 << 26)
    c, far = tensor(1 << 24, 2, 300), [1 << 32, 1 << 33, 1 << 34]
    assert L.load().flexatt_evict_rows(e, c, c, 1 << 27, kc, vc, *far, None) == -5


@pytest.mark.parametrize("which,on", [("scores", "key"), ("scores", "value"), ("slots", "scores"), ("slots", "key"),
                                      ("lengths", "slots"), ("lengths", "scores"), ("lengths", "value")])
def test_eviction_outputs_share_no_memory(which, on):
    at = dict(key=1 << 30, value=1 << 31, scores=1 << 32, slots=1 << 33, lengths=1 << 34)
    at[which] = at[on] + 4 * 100
    e = L.Evict(L.BF16, 2, 2, 300, 64, 100, 8, 4, 100, 0, 1 << 26)
    c = tensor(1 << 24, 2, 300)
    assert L.load().flexatt_evict_rows(e, c, c, 1 << 27, tensor(at["key"], 2, 100), tensor(at["value"], 2, 100),
                                       at["scores"], at["slots"], at["lengths"], None) == -5
