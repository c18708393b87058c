"""The rotary kernel's sine and cosine where their series are longest, next to an eighth of a turn."""
import math

import pytest
import torch

import flexatt_rotary as rot

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inter", [False, True])
def test_no_bias_next_to_an_eighth_of_a_turn(gpu_device, inter):
    """fp32 pairs (1, 0) at position 1 become (cos a, sin a) themselves.  Their mean error over 1024 angles: a series that
    ends too early is off to one side.  What may be: constants rounded, 2^-25 of the terms x^3 / 6 and x^4 / 24, under
    2.5e-9; three roundings of half steps 2^-25, standard deviation 3e-8, over 32 for the mean, four times that 4e-9;
    the terms left out 2e-9; 8.5e-9 in all (x^10 / 10! is 1.7e-8 at 0.76)."""
    f = torch.linspace(0.76, math.pi / 4 - 1e-4, 1024, dtype=torch.float64)
    x = torch.zeros(1, 1, 1, 256, device="cuda")
    first, second = (slice(0, 256, 2), slice(1, 256, 2)) if inter else (slice(0, 128), slice(128, 256))
    x[..., first] = 1.0
    pos = torch.ones(1, dtype=torch.int64, device="cuda")
    y = [rot.rotary_embedding(x, None, p.cuda(), positions=pos, interleaved=inter)[0][0, 0, 0].cpu().double()
         for p in f.chunk(8)]
    cos, sin = (torch.cat([z[part] for z in y]) for part in (first, second))
    for what, got, want in (("cos", cos, f.cos()), ("sin", sin, f.sin())):
        bias, worst = (got - want).mean().item(), (got - want).abs().max().item()
        assert abs(bias) <= 8.5e-9, f"{what}: mean error {bias:.2e}"
        assert worst <= 3.5 * 2.0 ** -24, f"{what}: {worst:.2e}"
