"""Attention over a cache of 8 bits, weight by weight: with a value of its own column for each key, an output is that key's
weight times its value, and for fp16 queries, whose weights are two numbers of fp16, exact to the output's rounding (on the
GPU, against the float64 oracle of oracle/cache_oracle.py)."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_tree import check, draw, tree

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16
F8, I8 = torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("dtype,D,T,n", [(FH, 128, 16, 100), (FH, 256, 16, 200), (FH, 64, 20, 40), (FH, 32, 9, 23), (BF, 128, 16, 100)])
def test_each_weight(gpu_device, dtype, D, T, n, kind, cap):
    """Sequences enough for some 10^5 weights; scales that differ by factors of e^4 and more."""
    B, Hq, Hkv, C = 12, 8, 2, n + T
    g = torch.Generator().manual_seed(D)
    q = draw(D, B, Hq, T, D, dtype)
    kc = torch.randint(-127, 128, (B, Hkv, C, D), generator=g).to(I8)
    kc = (kc if kind == I8 else kc.float().to(F8)).cuda()
    ks = torch.full((B, Hkv, C), 1 / 64, device="cuda")
    vs = torch.exp(2 * torch.randn(B, Hkv, C, generator=g)).cuda()
    vc = torch.zeros(B, Hkv, C, D)
    vc[:, :, torch.arange(C), torch.arange(C)] = 64.0
    vc = vc.to(kind).cuda()
    mask = tree(T, 3)[0]
    lengths = torch.full((B,), n, dtype=torch.int32)
    o = fc.quantized_tree_attention(q, kc, vc, ks, vs, lengths.cuda(), mask.cuda(), scale=0.02, soft_cap=cap)
    ro, _, to, _ = orc.quantized_tree_attention(*(x.cpu() for x in (q, kc, vc, ks, vs)), lengths, mask, scale=0.02, cap=cap,
                                                dtype=dtype)
    check("o", o, ro, to)
