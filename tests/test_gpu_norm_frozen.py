"""Gradients of norm and rotation where a part is frozen or not asked for: the rest are those of the whole pass (at these
sizes, which one workgroup a head has, bit by bit), and nothing is computed for a frozen query or key."""
import pytest
import torch

import flexatt_rotary as rot
from test_gpu_norm_rotary import weight
from test_gpu_rotary import draw

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
NAMES = ("q", "k", "wq", "wk")


def inputs(Hq=4, Hkv=2, S=33, D=64):
    f = rot.rotary_frequencies(D, device="cuda")[0]
    return dict(q=draw(1, 2, Hq, S, D, BF), k=draw(2, 2, Hkv, S, D, BF), wq=weight(3, D, BF), wk=weight(4, D, BF)), f, \
        (draw(5, 2, Hq, S, D, BF), draw(6, 2, Hkv, S, D, BF))


@pytest.mark.parametrize("asked", [m for m in range(1, 16)])
def test_parts_of_the_gradients(gpu_device, asked):
    x, f, g = inputs()
    names = [n for i, n in enumerate(NAMES) if asked >> i & 1]
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    whole = dict(zip(NAMES, torch.autograd.grad(rot.norm_rotary_embedding(*leaves.values(), f), list(leaves.values()), g)))
    y = rot.norm_rotary_embedding(*leaves.values(), f)  # all require them, some are asked for
    got = torch.autograd.grad(y, [leaves[n] for n in names], g)
    assert all(torch.equal(a, whole[n]) for a, n in zip(got, names))
    some = {n: t.clone().requires_grad_(n in names) for n, t in x.items()}  # some require them
    y = rot.norm_rotary_embedding(*some.values(), f)
    torch.autograd.backward(y, g)
    for n, t in some.items():
        assert torch.equal(t.grad, whole[n]) if n in names else t.grad is None
    if asked == 5:  # query and its weight without a key
        q, w = (x[n].clone().requires_grad_() for n in ("q", "wq"))
        y = rot.norm_rotary_embedding(q, None, w, None, f)[0]
        assert torch.equal(torch.autograd.grad(y, q, g[0], retain_graph=True)[0], whole["q"])
        assert torch.equal(torch.autograd.grad(y, w, g[0])[0], whole["wq"])


@pytest.mark.parametrize("frozen", ["k", "q"])
def test_no_memory_for_what_is_frozen(gpu_device, frozen):
    """The gradient of the frozen one would be 16 MB; its rows are the larger part."""
    x, f, g = inputs(*((1, 32) if frozen == "k" else (32, 1)), S=2048)
    for n in x:
        x[n].requires_grad_(not n.endswith(frozen))
    y = rot.norm_rotary_embedding(*x.values(), f)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    torch.autograd.backward(y, g)
    assert torch.cuda.max_memory_allocated() - before < 4 << 20
    assert all((t.grad is None) == n.endswith(frozen) for n, t in x.items())
