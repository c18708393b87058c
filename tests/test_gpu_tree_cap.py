"""The soft-capped LSE of tree attention, fp32 whatever the inputs' type, where few keys leave nothing to average."""
import pytest
import torch

import flexatt_cache as fc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top", [0.125, 12.0, 200.0])
@pytest.mark.parametrize("cap", [50.0, 7.0])
def test_lse_of_one_key(gpu_device, dtype, top, cap):
    """A drafted token alone sees itself: LSE is its capped score.  Queries and keys have one element, so the score s is
    exact.  In half steps h = 2^-24 of the capped score x: scale / cap 2, the quotient s / cap 1, the series 2, cap log2 e
    2, its product with tanh 1 and LSE in natural units 2, 10 in all; tanhf's own error, two steps, is 4 instead of 2; and 4
    h of 1 for 2^0 of the row sum, its logarithm and the sum of both.  Above |s| = cap / 4 (1 - 2 / (1 + e^2y)): 4 h of the
    cap more."""
    s = torch.linspace(-top, top, 301).to(dtype)
    q, k = torch.zeros(301, 1, 1, 64, dtype=dtype), torch.zeros(301, 1, 1, 64, dtype=dtype)
    q[..., 0], k[:, 0, 0, 0] = 1.0, s
    v = torch.randn(301, 1, 1, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    n = torch.zeros(301, dtype=torch.int32, device="cuda")
    o, lse = fc.tree_attention(q.cuda(), k.cuda(), v, n, scale=1.0, soft_cap=cap, return_lse=True)
    x = cap * torch.tanh(s.double() / cap)
    h = 2.0 ** -24
    tol = 12 * h * x.abs() + 4 * h + torch.where(s.double().abs() > 0.249 * cap, 4 * h * cap, 0.0)
    worst = ((lse[:, 0, 0].cpu().double() - x).abs() / tol).max().item()
    assert torch.equal(o, v)
    assert worst <= 1.0, f"{worst:.2f} tolerances"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lse_of_three_keys(gpu_device, dtype):
    """Two cached keys and the token itself, small scores of both signs: as above, of the largest score, with two more
    additions and the exponentials' steps (8 h of 1)."""
    g = torch.Generator().manual_seed(2)
    s = (torch.rand(400, 3, generator=g) - 0.5).to(dtype)
    q, k = torch.zeros(400, 1, 1, 128, dtype=dtype), torch.zeros(400, 1, 3, 128, dtype=dtype)
    q[..., 5], k[:, 0, :, 5] = 1.0, s
    n = torch.full((400,), 2, dtype=torch.int32, device="cuda")
    _, lse = fc.tree_attention(q.cuda(), k.cuda(), k.cuda(), n, scale=1.0, soft_cap=50.0, return_lse=True)
    x = 50.0 * torch.tanh(s.double() / 50.0)
    want, h = torch.logsumexp(x, dim=1), 2.0 ** -24
    tol = 12 * h * x.abs().amax(dim=1) + 2 * h * want.abs() + 12 * h
    worst = ((lse[:, 0, 0].cpu().double() - want).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.2f} tolerances"
