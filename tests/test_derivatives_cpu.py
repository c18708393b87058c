"""Derivatives that the rotary and cache calls cannot give are refused, not dropped.  The refusal comes before any other
check, so it is the same for CPU tensors and no kernel is launched here."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import flexatt_cache as fc
import flexatt_rotary as rot


def arguments():
    """Every call with its floating-point arguments by name."""
    x, c, n = torch.randn(1, 2, 3, 64), torch.randn(1, 2, 20, 64), torch.ones(1, dtype=torch.int32)
    f, s = torch.ones(32, dtype=torch.float64), torch.rand(1, 2, 20)
    out = [torch.zeros(1, 2, 9, 64), torch.zeros(1, 2, 9, 64), torch.zeros(1, 2, 9)]
    return {
        "rotary": (lambda a: rot.rotary_embedding(a["query"], a["key"], a["inv_freq"]),
                   dict(query=x, key=x, inv_freq=f)),
        "append": (lambda a: fc.rotary_append(a["query"], a["key"], a["value"], a["key_cache"], a["value_cache"], n,
                                              a["inv_freq"]),
                   dict(query=x, key=x, value=x, key_cache=c, value_cache=c, inv_freq=f)),
        "tree": (lambda a: fc.tree_attention(a["query"], a["key_cache"], a["value_cache"], n),
                 dict(query=x, key_cache=c, value_cache=c)),
        "weights": (lambda a: fc.attention_weight_sums(a["query"], a["key"], a["lse"], into=a["into"]),
                    dict(query=x, key=c, lse=torch.zeros(1, 2, 3), into=s)),
        "evict": (lambda a: fc.evict_cache(a["key_cache"], a["value_cache"], a["scores"], n, 9,
                                           out=(a["out key"], a["out value"], a["out scores"])),
                  dict(key_cache=c, value_cache=c, scores=s, **{"out key": out[0], "out value": out[1],
                                                                "out scores": out[2]})),
    }


EVERY = [(op, name) for op, (_, given) in arguments().items() for name in given]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op,name", EVERY)
def test_tangents_are_refused(op, name, grad):
    call, given = arguments()[op]
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        given[name] = fwd.make_dual(given[name], torch.ones_like(given[name]))
        with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
            call(given)
        given[name] = fwd.unpack_dual(given[name]).primal
        with pytest.raises(RuntimeError, match="ROCm GPU"):  # past the refusal
            call(given)


@pytest.mark.parametrize("op,name", [x for x in EVERY if x[0] != "rotary" or x[1] == "inv_freq"])
def test_gradients_are_refused(op, name):
    call, given = arguments()[op]
    given[name] = given[name].clone().requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
        call(given)
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm GPU"):  # past the refusal
        call(given)
