"""Keys and values side by side in one buffer, as the cache of an append and as the one that an eviction fills."""
import pytest
import torch

import flexatt_cache as fc

pytestmark = pytest.mark.gpu

B, H, C, D = 2, 3, 40, 64

LAYOUTS = {
    "rows": lambda x: (x.view(B, H, C, 2, D)[:, :, :, 0], x.view(B, H, C, 2, D)[:, :, :, 1]),
    "values first": lambda x: (x.view(B, H, C, 2, D)[:, :, :, 1], x.view(B, H, C, 2, D)[:, :, :, 0]),
    "tokens": lambda x: tuple(x.view(B, C, 2, H, D)[:, :, i].transpose(1, 2) for i in (0, 1)),
    "heads": lambda x: (x.view(B, 2, H, C, D)[:, 0], x.view(B, 2, H, C, D)[:, 1]),
    "halves": lambda x: (x.view(B, H, 2 * C, D)[:, :, :C], x.view(B, H, 2 * C, D)[:, :, C:]),
    "sequences": lambda x: (x.view(2, B, H, C, D)[0], x.view(2, B, H, C, D)[1]),
    "token by token": lambda x: tuple(x.view(C, 2, B, H, D)[:, i].permute(1, 2, 0, 3) for i in (0, 1)),
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_side_by_side(gpu_device, layout):
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    kc, vc = LAYOUTS[layout](new(2 * B * H * C * D))
    plain = kc.clone(memory_format=torch.contiguous_format), vc.clone(memory_format=torch.contiguous_format)
    q, k, v = new(B, 6, 5, D), new(B, H, 5, D), new(B, H, 5, D)
    n = torch.tensor([30, 2], dtype=torch.int32, device="cuda")
    fc.rotary_append(q, k, v, kc, vc, n, None)
    fc.rotary_append(q, k, v, *plain, n, None)
    assert torch.equal(kc, plain[0]) and torch.equal(vc, plain[1])
    big, scores = (new(B, H, 90, D), new(B, H, 90, D)), torch.rand(B, H, 90, generator=g, device="cuda")
    m = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    want = fc.evict_cache(*big, scores, m, 37, recent=3)
    got = fc.evict_cache(*big, scores, m, 37, recent=3, out=(kc, vc, torch.zeros(B, H, C, device="cuda")))
    for b, x in enumerate(want[4].tolist()):
        assert torch.equal(got[0][b, :, :x], want[0][b, :, :x]) and torch.equal(got[1][b, :, :x], want[1][b, :, :x])
        assert torch.equal(kc[b, :, x:], plain[0][b, :, x:]) and torch.equal(vc[b, :, x:], plain[1][b, :, x:])
    assert torch.equal(got[3], want[3]) and torch.equal(got[4], want[4])
