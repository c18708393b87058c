"""Attention over a cache of 8 bits: the value scales of rows that a token does not see, whatever they are, leave its result
as it is (on the GPU, against the float64 oracle of oracle/cache_oracle.py and bit by bit)."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_quant_tree import cache
from test_gpu_tree import check, draw

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16
F8, I8 = torch.float8_e4m3fn, torch.int8
ODD = [2.0 ** 60, 3e38, float("inf"), float("nan")]


def setup(dtype, kind, D, T, C, seed=0):
    q = draw(seed, 1, 4, T, D, dtype)
    (kc, ks), (vc, vs) = cache(seed + 2, 1, 2, C, D, kind), cache(seed + 3, 1, 2, C, D, kind)
    return q, kc, vc, ks, vs


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("dtype,kind,D", [(BF, F8, 128), (FH, I8, 128), (BF, I8, 64), (FH, F8, 64), (BF, F8, 256), (FH, I8, 32)])
def test_a_drafted_token_that_the_others_do_not_see(gpu_device, dtype, kind, D, odd):
    """Token 1's value is odd; the others see all but it: their results are those of an ordinary scale in its place."""
    T, n = 5, 70
    q, kc, vc, ks, vs = setup(dtype, kind, D, T, 90)
    mask = torch.ones(T, T, dtype=torch.bool).tril()
    mask[:, 1] = False
    mask[1, 1] = True
    lengths = torch.tensor([n], dtype=torch.int32)
    vs[:, :, n + 1] = 1.0
    ro, rl, to, tl = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), lengths, mask, dtype=dtype)
    vs[:, :, n + 1] = odd
    o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths.cuda(), mask.cuda(), return_lse=True)
    others = [0, 2, 3, 4]
    check("o", o[:, :, others], ro[:, :, others], to[:, :, others])
    check("lse", lse, rl, tl)
    if odd == 2.0 ** 60 and dtype == BF:  # and the token that sees it
        ro, _, to, _ = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), lengths, mask, dtype=dtype)
        check("o", o[:, :, 1:2], ro[:, :, 1:2], to[:, :, 1:2])


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("T", [1, 12])
def test_rows_before_a_window(gpu_device, T, odd):
    """Rows of the tiles that a window begins in, and each token's own rows before it."""
    n, window = 400, 90
    q, kc, vc, ks, vs = setup(BF, F8, 128, T, 450)
    lengths = torch.tensor([n], dtype=torch.int32)
    want = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths.cuda(), sliding_window=window, return_lse=True)
    vs[:, :, :n - window] = odd
    got = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths.cuda(), sliding_window=window, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    vs[:, :, :n - window] = 1.0
    vs[:, :, n - window] = odd  # seen by token 0 alone
    got = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths.cuda(), sliding_window=window, return_lse=True)
    vs[:, :, n - window] = 1.0
    ro, rl, to, tl = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), lengths, window=window)
    check("lse", got[1], rl, tl)
    if T > 1:
        check("o", got[0][:, :, 1:], ro[:, :, 1:], to[:, :, 1:])


def test_rows_that_nobody_sees(gpu_device):
    """A drafted token that no token sees, itself included."""
    q, kc, vc, ks, vs = setup(FH, I8, 64, 6, 500)
    lengths = torch.tensor([430], dtype=torch.int32, device="cuda")
    mask = torch.ones(6, 6, dtype=torch.bool, device="cuda").tril()
    mask[:, 3] = False
    want = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths, mask, return_lse=True)
    for odd in ODD:
        vs[:, :, 433] = odd
        got = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths, mask, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
