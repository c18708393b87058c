"""Function transforms of the rotary and cache calls on the GPU: refused, where they would lose a derivative."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import flexatt_cache as fc
import flexatt_rotary as rot

pytestmark = pytest.mark.gpu


def test_forward_mode_and_transforms_are_refused(gpu_device):
    q = torch.randn(2, 2, 5, 64, device="cuda")
    c, n = torch.randn(2, 2, 20, 64, device="cuda"), torch.tensor([4, 9], dtype=torch.int32, device="cuda")
    f, _ = rot.rotary_frequencies(64, device="cuda")
    for call in (lambda x: rot.rotary_embedding(x, None, f)[0], lambda x: fc.tree_attention(x, c, c, n)):
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                call(fwd.make_dual(q, torch.ones_like(q)))
            plain = call(fwd.unpack_dual(fwd.make_dual(q, torch.ones_like(q))).primal)
        assert torch.equal(plain, call(q))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x: call(x).sum())(q)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(q[None])
