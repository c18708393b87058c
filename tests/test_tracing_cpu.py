"""A trace through a rotary or cache call would hold its outputs' memory and not the kernel that fills it: refused, before
any other check."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import flexatt_cache as fc
import flexatt_rotary as rot

CALLS = {
    "rotary": lambda x, c, n, f, s: rot.rotary_embedding(x, x, f)[0],
    "append": lambda x, c, n, f, s: fc.rotary_append(x, x, x, c, c + 1, n, f),
    "tree": lambda x, c, n, f, s: fc.tree_attention(x, c, c, n),
    "weights": lambda x, c, n, f, s: fc.attention_weight_sums(x, c, x[..., 0]),
    "evict": lambda x, c, n, f, s: fc.evict_cache(c, c, s, n, 9)[0],
}


def arguments():
    return (torch.randn(1, 2, 3, 64), torch.randn(1, 2, 20, 64), torch.ones(1, dtype=torch.int32),
            torch.ones(32, dtype=torch.float64), torch.rand(1, 2, 20))


class Watching(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("op", CALLS)
def test_traces_are_refused(op):
    a = arguments()
    for mode in ("real", "fake"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(CALLS[op], tracing_mode=mode)(*a)
    with FakeTensorMode(allow_non_fake_inputs=True) as fake:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            CALLS[op](*(fake.from_tensor(t) for t in a))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(CALLS[op], a)
    with Watching(), pytest.raises(RuntimeError, match="ROCm GPU"):  # a mode that only looks on
        CALLS[op](*a)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        CALLS[op](*a)
