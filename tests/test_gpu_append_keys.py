"""Keys and values put into a cache without a query, as a prompt's keys for later queries."""
import pytest
import torch

import flexatt_cache as fc
import flexatt_rotary as rot

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,pairs", [(64, 32), (128, 9)])  # both kernels
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_without_query_heads(gpu_device, D, pairs, dtype):
    g = torch.Generator().manual_seed(1)
    new = lambda h, s: torch.randn(2, h, s, D, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v, kc, vc = new(4, 7), new(2, 7), new(2, 7), new(2, 30), new(2, 30)
    n, f = torch.tensor([3, 25], dtype=torch.int32, device="cuda"), rot.rotary_frequencies(2 * pairs, device="cuda")[0]
    want = kc.clone(), vc.clone()
    fc.rotary_append(q, k, v, *want, n, f)
    before = kc._version, vc._version
    y = fc.rotary_append(q[:, :0], k, v, kc, vc, n, f)
    assert y.shape == (2, 0, 7, D) and y.dtype == dtype
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    assert kc._version > before[0] and vc._version > before[1]
    assert fc.rotary_append(q[:, :0, :0], k[:, :, :0], v[:, :, :0], kc, vc, n, f).shape == (2, 0, 0, D)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
