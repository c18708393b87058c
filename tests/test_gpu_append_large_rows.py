"""Keys whose squares pass 32 bits, normalised on the way into a cache of 8 bits, on the GPU against the float64 oracle
(oracle/cache_oracle.py): what decides their codes is in 64 bits, and the normalised row is one of ordinary size."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc
from test_gpu_norm_rotary import weight
from test_gpu_quant_cache import caches, nearest
from test_gpu_rotary import draw

pytestmark = pytest.mark.gpu

BF, FS = torch.bfloat16, torch.float32
F8, I8 = torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("pairs", [64, 9])
@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("dtype", [BF, FS])
def test_codes_of_large_rows(gpu_device, dtype, kind, pairs):
    """Rows of sizes 2^60 to 2^125 among ordinary and small ones.  The bounds are those of ordinary rows (see
    test_gpu_quant_cache.test_codes_at_borders): 64 bits leave 1e-11 of a row's largest size."""
    B, H, S, D = 1, 3, 60, 128
    k = draw(5, B, H, S, D, dtype)
    k *= torch.exp2(torch.tensor([0, 60, 63, 64, 66, 90, 124, -20, 65, -60])[torch.arange(S) % 10].float()).to(dtype).cuda()[:, None]
    k[0, 1, 7::20] = 0
    f, w = rot.rotary_frequencies(2 * pairs, device="cuda")[0], weight(4, D, FS)
    kc, vc, ks, vs = caches(3, B, H, S, D, kind)
    fc.quantized_append(k[:, :0], k, k, kc, vc, ks, vs, torch.zeros(B, dtype=torch.int32, device="cuda"), f,
                        query_weight=w, key_weight=w, eps=1e-6)
    y, _ = orc.norm_rotary(k.cpu().double(), w.cpu().double(), f.cpu(), torch.arange(S).expand(B, S), False, 1.0,
                           float(torch.tensor(1e-6)))
    size = y.abs().amax(dim=-1).clamp(min=2.0 ** -100) / orc.TOP[kind]
    assert bool(((ks.cpu().double() - size).abs() <= size * (2.0 ** -24 + 2e-11)).all())
    once = 2.0 ** -19 if kind == F8 else 0.0
    assert nearest(y, ks.cpu().double(), kc.cpu(), kind) <= 1.0 + once + 1e-11 * (448 * 2 ** 10 if kind == F8 else 127 * 2)
