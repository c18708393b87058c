"""Heads whose squares pass 32 bits, normalised and turned, and the gradients, on the GPU against the float64 oracle
(oracle/cache_oracle.py): the bounds are those of ordinary rows."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot
from oracle import cache_oracle as orc
from test_gpu_norm_rotary import weight
from test_gpu_rotary import draw, within

pytestmark = pytest.mark.gpu

BF, FS = torch.bfloat16, torch.float32

# powers of two by which rows are larger
SIZES = torch.tensor([0, 60, 63, 64, 66, 90, 124, -10, 65, 2])


@pytest.mark.parametrize("pairs,inter", [(64, False), (64, True), (9, False), (0, False)])
@pytest.mark.parametrize("dtype", [BF, FS])
def test_large_rows(gpu_device, dtype, pairs, inter):
    B, Hq, Hkv, S, D, eps = 2, 5, 2, 70, 128, 1e-5
    up = torch.exp2(SIZES[torch.arange(S) % 10].float()).to(dtype).cuda()[:, None]
    q, k = draw(1, B, Hq, S, D, dtype) * up, draw(2, B, Hkv, S, D, dtype) * up.flip(0)
    wq, wk = weight(3, D, FS), weight(4, D, FS)
    gq, gk = draw(5, B, Hq, S, D, dtype), draw(6, B, Hkv, S, D, dtype)
    f = rot.rotary_frequencies(2 * pairs, device="cuda")[0] if pairs else torch.empty(0, dtype=torch.float64, device="cuda")
    for x in (q, k, wq, wk):
        x.requires_grad_()
    y = rot.norm_rotary_embedding(q, k, wq, wk, f, interleaved=inter, eps=eps)
    d = torch.autograd.grad(y, (q, wq, k, wk), (gq, gk))
    at, eps = torch.arange(S).expand(B, S), float(torch.tensor(eps))
    for x, w, g, out, dx, dw, name in ((q, wq, gq, y[0], d[0], d[1], "q"), (k, wk, gk, y[1], d[2], d[3], "k")):
        x, w, g = (t.detach().cpu().double() for t in (x, w, g))
        ref, slack = orc.norm_rotary(x, w, f.cpu(), at, inter, 1.0, eps)
        within(out, ref, orc.rounded(ref, slack, dtype), name)
        (rx, sx), (rw, sw) = orc.norm_rotary_grad(x, w, g, f.cpu(), at, inter, 1.0, eps)
        # (dx of the largest rows are about the smallest numbers of 32 bits, under which a result may be 0)
        within(dx, rx, orc.rounded(rx, sx, dtype) + 2.0 ** -126, "d" + name)
        within(dw, rw, orc.rounded(rw, sw, FS), "dw" + name)


@pytest.mark.parametrize("dtype", [BF, FS])
def test_rows_of_the_largest_numbers_and_no_numbers(gpu_device, dtype):
    """Rows of the type's largest number are rows of ones; an infinity or NaN makes NaN of its own row's elements, no other
    row changes, on the way into a cache too."""
    x = draw(1, 1, 4, 8, 64, dtype)
    x[0, 0, 1] = torch.finfo(dtype).max
    x[0, 1, 2, 1::2] = -torch.finfo(dtype).max
    x[0, 1, 2, ::2] = torch.finfo(dtype).max
    one = torch.ones(64, device="cuda")
    good = rot.norm_rotary_embedding(x, None, one, None, torch.empty(0, dtype=torch.float64, device="cuda"))[0]
    want = torch.ones(64)
    assert bool(((good[0, 0, 1].float().cpu() - want).abs() <= 2.0 ** -7).all())
    want[1::2] = -1
    assert bool(((good[0, 1, 2].float().cpu() - want).abs() <= 2.0 ** -7).all())
    x[0, 2, 3, 5] = float("inf")
    x[0, 2, 4, 5] = float("nan")
    f = torch.empty(0, dtype=torch.float64, device="cuda")
    y = rot.norm_rotary_embedding(x, None, one, None, f)[0]
    assert bool(torch.isnan(y[0, 2, 3, 5])) and bool(torch.isnan(y[0, 2, 4]).all())
    rest = torch.ones(1, 4, 8, dtype=torch.bool)
    rest[0, 2, 3:5] = False
    assert torch.equal(y.cpu()[rest], good.cpu()[rest])
    kc, vc = torch.zeros(2, 1, 4, 8, 64, dtype=dtype, device="cuda")
    q = fc.norm_rotary_append(x, x, x, kc, vc, torch.zeros(1, dtype=torch.int32, device="cuda"), one, one, f)
    assert torch.equal(q.cpu()[rest], good.cpu()[rest]) and torch.equal(kc.cpu()[rest], good.cpu()[rest])
