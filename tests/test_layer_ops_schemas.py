"""The operators keep to their schemas: what they write is marked, what they return shares no memory with an argument."""
import pytest
import torch

import _lib

bf, dev = torch.bfloat16, "cuda"
NAMES = ["deltanet_chunk", "deltanet_step", "gated_norm", "norm_residual"]


@pytest.mark.parametrize("name", NAMES)
def test_schema_returns_alias_nothing(name):
    schema = getattr(_lib.ops(), name).default._schema
    assert all(r.alias_info is None for r in schema.returns)
    written = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert written == {"deltanet_chunk": {"final_state", "out"}, "deltanet_step": {"out_state", "out"}, "gated_norm": set(),
                       "norm_residual": {"out"}}[name]


def calls():
    T, H, Hk, d = 12, 4, 2, 64
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)

    def rnd(*shape, dtype=bf):
        return torch.randn(*shape, device=dev, generator=gen).to(dtype)

    q, k, v = rnd(1, T, Hk, d), rnd(1, T, Hk, d), rnd(1, T, H, d)
    g, b = -rnd(1, T, H, dtype=torch.float32).abs(), torch.sigmoid(rnd(1, T, H))
    cu = torch.tensor([0, 5, T], dtype=torch.int32, device=dev)
    S, S2, out = rnd(2, H, d, d, dtype=torch.float32), rnd(2, H, d, d, dtype=torch.float32), torch.zeros_like(v)
    for s1 in (None, S2):
        for o in (None, out):
            yield "deltanet_chunk", (q, k, v, g, b, cu, S, s1, o)
    pool, pool2 = rnd(T, H, d, d, dtype=torch.float32), torch.zeros(T, H, d, d, device=dev)
    index = torch.arange(T, dtype=torch.int32, device=dev).flip(0)
    for o in (None, out[0]):
        yield "deltanet_step", (q[0], k[0], v[0], g[0], b[0], pool, index, pool2, o)
    w = rnd(d)
    yield "gated_norm", (v[0], rnd(T, H, d), w, 1e-6)
    block, residual, w = rnd(T, H * d), rnd(T, H * d), rnd(H * d)
    for nxt in (None, w):
        for o in (None, torch.zeros_like(residual)):
            yield "norm_residual", (block, residual, w, None, True, 1.0, nxt, 1e-6, o)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(11))
def test_operator_keeps_to_its_schema(i):
    name, args = list(calls())[i]
    f = getattr(_lib.ops(), name).default
    torch.library.opcheck(f, args, test_utils="test_schema")
    got = f(*args)
    got = [t.untyped_storage().data_ptr() for t in (got if isinstance(got, tuple) else (got,)) if t.numel()]
    taken = {t.untyped_storage().data_ptr() for t in args if isinstance(t, torch.Tensor)}
    assert len(set(got)) == len(got) and not taken & set(got)


@pytest.mark.gpu
def test_given_tensors_are_returned_by_the_wrappers():
    import deltanet
    import norms
    every = list(calls())
    for name, a in every:
        if name == "deltanet_chunk":
            o, S = deltanet.chunk_gated_delta_rule(*a[:5], initial_state=a[6], cu_seqlens=a[5], final_state=a[7], out=a[8])
            assert (o is a[8] or a[8] is None) and (S is a[7] or a[7] is None)
            assert o.shape == a[2].shape and S.shape == a[6].shape
        elif name == "deltanet_step":
            o, S = deltanet.step_gated_delta_rule(*a[:6], state_index=a[6], out_state=a[7], out=a[8])
            assert S is a[7] and (o is a[8] or a[8] is None) and o.shape == a[2].shape
        elif name == "norm_residual":
            r, n = norms.norm_residual(a[0], a[1], a[2], next_weight=a[6], out=a[8])
            assert (r is a[8] or a[8] is None) and r.shape == a[1].shape and (n is None) == (a[6] is None)
