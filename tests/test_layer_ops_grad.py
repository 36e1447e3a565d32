"""The forward-only operators refuse a tensor that requires a gradient while gradients are recorded."""
import pytest
import torch

import deltanet
import norms

bf = torch.bfloat16


def rows(dev, T=3, H=2, d=64):
    return [torch.zeros(T, H, d, dtype=bf, device=dev) for _ in range(3)] + [torch.zeros(T, H, device=dev),
                                                                            torch.zeros(T, H, dtype=bf, device=dev)]


def calls(dev):
    """name of each operand -> (its tensor, the call)"""
    T, H, d = 3, 2, 64
    x = rows(dev)
    S, S1 = torch.zeros(1, H, d, d, device=dev), torch.zeros(1, H, d, d, device=dev)
    out = torch.zeros(1, T, H, d, dtype=bf, device=dev)
    f = lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), initial_state=S, final_state=S1, out=out)
    for name, t in zip(("query", "key", "value", "g", "beta", "initial_state", "final_state", "out"), (*x, S, S1, out)):
        yield name, t, f
    y = rows(dev)
    pool, pool1, o = torch.zeros(T, H, d, d, device=dev), torch.zeros(T, H, d, d, device=dev), out[0].clone()
    f2 = lambda: deltanet.step_gated_delta_rule(*y, pool, out_state=pool1, out=o)
    for name, t in zip(("query", "key", "value", "g", "beta", "state", "out_state", "out"), (*y, pool, pool1, o)):
        yield name, t, f2
    a, b, w = (torch.zeros(T, H, d, dtype=bf, device=dev), torch.zeros(T, H, d, dtype=bf, device=dev),
               torch.zeros(d, dtype=bf, device=dev))
    f3 = lambda: norms.gated_rms_norm(a, b, w)
    for name, t in (("x", a), ("z", b), ("weight", w)):
        yield name, t, f3
    n = [torch.zeros(T, d, dtype=bf, device=dev) for _ in range(3)] + [torch.zeros(d, device=dev) for _ in range(2)]
    r = torch.zeros(T, d, dtype=bf, device=dev)
    f4 = lambda: norms.norm_residual(n[0], n[1], gate=n[2], post_weight=n[3], next_weight=n[4], out=r)
    for name, t in zip(("block", "residual", "gate", "post_weight", "next_weight", "out"), (*n, r)):
        yield name, t, f4


COUNT = 25


def check(i, dev):
    every = list(calls(dev))
    assert len(every) == COUNT
    name, t, f = every[i]
    t.requires_grad_()
    with pytest.raises(RuntimeError, match=f"is forward only and {name} requires a gradient"):
        f()
    return f


@pytest.mark.parametrize("i", range(COUNT))
def test_refused(i):
    check(i, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(COUNT))
def test_refused_and_taken_without_gradients(i):
    f = check(i, "cuda")
    with torch.no_grad():
        f()
