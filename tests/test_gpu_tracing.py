"""Rotary and cache calls in compiled functions, and traces that would leave them out."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import flexatt_cache as fc
import flexatt_rotary as rot

pytestmark = pytest.mark.gpu


def test_a_compiled_function_runs_the_calls_as_they_are(gpu_device):
    q = torch.randn(1, 4, 3, 64, device="cuda")
    k, v = torch.randn(1, 2, 3, 64, device="cuda"), torch.randn(1, 2, 3, 64, device="cuda")
    n, f = torch.tensor([5], dtype=torch.int32, device="cuda"), rot.rotary_frequencies(64, device="cuda")[0]

    def step(q, k, v, kc, vc):
        q = fc.rotary_append(q * 2.0, k, v + 1.0, kc, vc, n, f)
        return fc.tree_attention(q, kc, vc, n) * 0.5

    caches = [torch.randn(1, 2, 20, 64, device="cuda") for _ in range(2)]
    want_caches = [c.clone() for c in caches]
    want = step(q, k, v, *want_caches)
    got = torch.compile(step, backend="aot_eager")(q, k, v, *caches)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(caches, want_caches))


def test_a_traced_backward_pass_is_refused(gpu_device):
    q = torch.randn(1, 4, 3, 64, device="cuda", requires_grad=True)
    y, _ = rot.rotary_embedding(q, None, rot.rotary_frequencies(64, device="cuda")[0])
    g = torch.randn_like(y)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(y, q, g, retain_graph=True)[0])(g)
    assert torch.autograd.grad(y, q, g)[0].shape == q.shape
