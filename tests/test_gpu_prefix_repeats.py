"""Attention behind a shared prefix with eight row tiles a workgroup, whose running maximum reads MFMA results in asm, where
the wait states are the source's to keep: the same call, with other work between the repetitions, gives the same bits."""
import pytest
import torch

import flexatt_cache as fc
from test_gpu_tree import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_repeats_after_other_work(gpu_device, dtype, cap):
    q, kc, vc = draw(1, 64, 16, 1, 128, dtype), draw(2, 64, 2, 40, 128, dtype), draw(3, 64, 2, 40, 128, dtype)
    pk, pv = draw(4, 1, 2, 2100, 128, dtype)[0], draw(5, 1, 2, 2100, 128, dtype)[0]
    q2, pk2 = draw(6, 64, 16, 1, 128, dtype, spread=4.0), draw(7, 1, 2, 2100, 128, dtype, spread=4.0)[0]
    n = (torch.arange(64, dtype=torch.int32) % 39).cuda()
    first = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, soft_cap=cap, return_lse=True)
    for _ in range(6):
        fc.shared_prefix_attention(q2, pk2, pv, kc, vc, n, soft_cap=cap)
        torch.matmul(torch.randn(256, 256, device="cuda"), torch.randn(256, 256, device="cuda"))
        again = fc.shared_prefix_attention(q, pk, pv, kc, vc, n, soft_cap=cap, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
