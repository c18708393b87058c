"""Attention behind a shared prefix: the error's rms beside that of rounding the exact result to the type.  Where a wave has a
row tile alone the weights lose nothing, elsewhere they are rounded once."""
import pytest
import torch

import flexatt_cache as fc
from oracle import cache_oracle as orc
from test_gpu_tree import draw

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("B,Hq,Hkv,T,P,C,D,most", [
    (8, 8, 2, 1, 2048, 300, 128, 1.03), (2, 4, 1, 2, 5000, 700, 64, 1.03), (3, 4, 2, 1, 700, 40, 32, 1.03),
    (3, 8, 2, 11, 1500, 300, 256, 1.03),                                                # a row tile alone at any size
    (5, 8, 1, 2, 3000, 200, 128, 1.45), (6, 7, 1, 4, 2000, 200, 64, 1.45), (64, 8, 1, 1, 2000, 40, 128, 1.45)])
def test_error_beside_the_outputs_rounding(gpu_device, dtype, cap, B, Hq, Hkv, T, P, C, D, most):
    q, kc, vc = draw(1, B, Hq, T, D, dtype), draw(2, B, Hkv, C, D, dtype), draw(3, B, Hkv, C, D, dtype)
    pk, pv = draw(4, 1, Hkv, P, D, dtype)[0], draw(5, 1, Hkv, P, D, dtype)[0]
    n = torch.tensor([(C - T) * (b + 1) // B for b in range(B)], dtype=torch.int32)
    o = fc.shared_prefix_attention(q, pk, pv, kc, vc, n.cuda(), soft_cap=cap).cpu().double()
    ref = orc.prefix_attention(*(x.cpu() for x in (q, pk, pv, kc, vc)), n, cap=cap, dtype=dtype)[0]
    rms = lambda x: x.square().mean().sqrt().item()  # noqa: E731
    assert rms(o - ref) <= most * rms(ref.to(dtype).double() - ref)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D,P,T,n", [(128, 70, 3, 50), (64, 40, 2, 20), (256, 150, 4, 90), (32, 17, 1, 12)])
def test_each_weight(gpu_device, dtype, cap, D, P, T, n):
    """A value of its own column for each key: an output is that key's weight, which has lost nothing but the output's
    rounding."""
    B, Hq, Hkv, C = 2, 8, 2, n + T
    q, kc, pk = draw(1, B, Hq, T, D, dtype), draw(2, B, Hkv, C, D, dtype), draw(3, 1, Hkv, P, D, dtype)[0]
    pv, vc = torch.zeros(Hkv, P, D), torch.zeros(B, Hkv, C, D)
    pv[:, torch.arange(P), torch.arange(P)] = 1.0
    vc[:, :, torch.arange(C), P + torch.arange(C)] = 1.0
    pv, vc = pv.to(dtype).cuda(), vc.to(dtype).cuda()
    lengths = torch.full((B,), n, dtype=torch.int32)
    o = fc.shared_prefix_attention(q, pk, pv, kc, vc, lengths.cuda(), soft_cap=cap)
    ref, _, _, _ = orc.prefix_attention(*(x.cpu() for x in (q, pk, pv, kc, vc)), lengths, cap=cap, dtype=dtype)
    eps = torch.finfo(dtype).eps  # half a step, and scores' errors of some 2^-16 each
    least = 2.0 ** -24 if dtype == FH else 0.0
    assert bool(((o.cpu().double() - ref).abs() <= ref * (eps / 2 + 2.0 ** -14) + least).all())
