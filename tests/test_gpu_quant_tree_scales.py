"""Attention over a cache of 8 bits whose values differ in size by more than 32 bits hold, on the GPU against the float64
oracle (oracle/cache_oracle.py): a row's sum of weights does not depend on the values' scales."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_quant_tree import cache
from test_gpu_tree import check, draw

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16
F8, I8 = torch.float8_e4m3fn, torch.int8


def against_oracle(q, kc, ks, vc, vs, n, **kw):
    n = torch.tensor(n, dtype=torch.int32)
    o, lse = fc.quantized_tree_attention(q, kc, vc, ks, vs, n.cuda(), return_lse=True, **kw)
    ro, rl, to, tl = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), n, dtype=q.dtype)
    check("o", o, ro, to)
    check("lse", lse, rl, tl)


@pytest.mark.parametrize("power", [40, 75, 100, 118])
@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_zeros_and_large_values(gpu_device, D, kind, power):
    """Value rows of zeros, whose scale is the smallest, and rows about 2^power: the former first, last, in turns of a tile
    (so that some waves meet one kind alone) and of a row."""
    C = 1100
    q = draw(1, 1, 4, 2, D, BF, spread=0.3)
    (kc, ks), (vc, vs) = cache(2, 1, 2, C, D, kind), cache(3, 1, 2, C, D, kind)
    j = torch.arange(C, device="cuda")
    for zero in (j < C // 2, j >= C // 2, j // 32 % 2 == 0, j // 32 % 2 == 1, j // 32 % 4 != 1, j % 2 == 0, j < C - 1):
        c = torch.where(zero[:, None], torch.zeros_like(vc.view(torch.uint8)), vc.view(torch.uint8)).view(kind)
        s = torch.where(zero, torch.full_like(vs, 2.0 ** -100 / orc.TOP[kind]), vs * 2.0 ** power)
        against_oracle(q, kc, ks, c, s, [C - 2])


@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_smallest_and_largest_scales(gpu_device, D, kind):
    """All scales about 2^power, down to the smallest that is written; growing and shrinking along the cache."""
    C = 700
    q = draw(1, 1, 4, 2, D, BF)
    (kc, ks), (vc, vs) = cache(2, 1, 2, C, D, kind), cache(3, 1, 2, C, D, kind)
    unit = vs / vs.log2().mean().exp2()
    for power in (-108, -100, -84, -60, -33, 33, 60, 100, 114):
        against_oracle(q, kc, ks, vc, unit * 2.0 ** power, [C - 2])
    ramp = torch.linspace(-105, 110, C, device="cuda").exp2()
    for s in (ramp, ramp.flip(0)):
        against_oracle(q, kc, ks, vc, s.expand(1, 2, C).contiguous(), [C - 2])


@pytest.mark.parametrize("i", range(4))
def test_error_is_the_outputs_rounding(gpu_device, i):
    """fp16 and bf16: the error's rms is that of rounding the result alone (one fp16 operand for the weights would make it
    1.3 times as much for fp16)."""
    dtype, kind, D, T = ((FH, F8, 128, 16), (FH, I8, 64, 40), (FH, I8, 256, 3), (BF, F8, 128, 16))[i]
    q = draw(1, 2, 8, T, D, dtype)
    (kc, ks), (vc, vs) = cache(2, 2, 2, 3500, D, kind), cache(3, 2, 2, 3500, D, kind, 0.6)
    n = torch.tensor([3400, 1700], dtype=torch.int32)
    o = fc.quantized_tree_attention(q, kc, vc, ks, vs, n.cuda()).cpu().double()
    ro, _, to, _ = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), n, dtype=dtype)
    rms = lambda x: x.square().mean().sqrt().item()  # noqa: E731
    assert rms(to) < rms(ro) / 8
    assert rms(o - ro) <= 1.1 * rms(ro.to(dtype).double() - ro)
