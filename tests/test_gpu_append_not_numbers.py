"""Keys that become NaN or infinite on the way into a cache of 8 bits, by a weight or a frequency, on the GPU: such a row
has codes of 0 and a scale of NaN, whatever it was before."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from test_gpu_norm_rotary import weight
from test_gpu_quant_cache import bits, caches
from test_gpu_rotary import draw

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
F8, I8 = torch.float8_e4m3fn, torch.int8
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("what", ["one weight", "all weights", "infinite weight", "infinite weight of zeros", "frequency",
                                  "infinite frequency", "infinite frequency, one of the places"])
@pytest.mark.parametrize("pairs", [32, 5])
@pytest.mark.parametrize("kind", [F8, I8])
@pytest.mark.parametrize("dtype", [BF, FH, FS])
def test_rows_that_become_no_numbers(gpu_device, dtype, kind, pairs, what):
    B, H, S, D = 2, 2, 9, 64
    q, k, v = draw(1, B, 2 * H, S, D, dtype), draw(2, B, H, S, D, dtype), draw(3, B, H, S, D, dtype)
    f, w = rot.rotary_frequencies(2 * pairs, device="cuda")[0], weight(4, D, FS)
    good, norm = weight(4, D, FS), dict(eps=1e-5)
    if "weight" in what:
        at = slice(None) if what == "all weights" else 37
        w[at] = INF if "infinite" in what else NAN
        if what == "infinite weight of zeros":
            k[..., 37] = 0
        norm.update(query_weight=good, key_weight=w)
    else:
        f[3] = INF if "infinite" in what else NAN
    start = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    pos = None
    if what.endswith("places"):  # an angle of 0 times infinity, and of infinity
        pos = torch.arange(S, device="cuda")
    kc, vc, ks, vs = caches(7, B, H, S + 6, D, kind)
    kc2, vc2, ks2, vs2 = (x.clone() for x in (kc, vc, ks, vs))
    fc.quantized_append(q, k, v, kc, vc, ks, vs, start, f, positions=pos, **norm)
    fc.quantized_append(q, k, v, kc2, vc2, ks2, vs2, start, None)  # (what becomes of the values)
    new = torch.zeros(B, S + 6, dtype=torch.bool)
    for b, n in enumerate(start.tolist()):
        new[b, n:n + S] = True
    new = new[:, None].expand(B, H, S + 6)
    assert bool((bits(kc).cpu()[new] == 0).all()) and bool(torch.isnan(ks.cpu()[new]).all())
    assert not bool(torch.isnan(ks.cpu()[~new]).any())
    assert torch.equal(bits(vc), bits(vc2)) and torch.equal(vs, vs2)


@pytest.mark.parametrize("kind", [F8, I8])
def test_only_the_rows_it_happens_to(gpu_device, kind):
    """Positions that a frequency of 1e300 takes beyond 64 bits, for two of the tokens."""
    k = draw(2, 1, 2, 6, 64, BF)
    f = rot.rotary_frequencies(64, device="cuda")[0]
    f[0] = 1e300
    pos = torch.tensor([0, 1 << 62, 0, 0, -(1 << 62), 0], device="cuda")
    kc, vc, ks, vs = caches(7, 1, 2, 6, 64, kind)
    fc.quantized_append(k[:, :0], k, k, kc, vc, ks, vs, torch.zeros(1, dtype=torch.int32, device="cuda"), f, positions=pos)
    bad = torch.tensor([False, True, False, False, True, False])
    assert torch.equal(torch.isnan(ks[0]).cpu(), bad.expand(2, 6)) and not bool(torch.isnan(vs).any())
    assert bool((bits(kc)[0].cpu()[:, bad] == 0).all()) and torch.equal(bits(kc)[0][:, ~bad], bits(vc)[0][:, ~bad])
