"""Host-side refusals of the batched delta rule and the norms, without a GPU."""
import ctypes

import pytest
import torch

import _lib
import deltanet
import norms

FAKE, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10008)
FAR = ctypes.c_void_p(0x7f0000000000)
STRIDES = (ctypes.c_int64 * 10)(*([128] * 10))


def step(q=FAKE, strides=STRIDES, index=FAKE, slots=4, s_in=FAKE, s_out=FAR, out=FAKE, rows=2, H=4, Hk=2, dk=128, dv=128):
    return _lib.lib().qfn_deltanet_step_batch(q, FAKE, FAKE, FAKE, FAKE, strides, index, slots, s_in, s_out, out, rows, H,
                                              Hk, dk, dv, None)


def test_step_refusals():
    assert step(q=None) == 1 and step(out=None) == 1 and step(strides=None) == 1
    assert step(s_in=None) == 1 and step(s_out=None) == 1
    assert step(H=4, Hk=3) == 1 and step(H=0) == 1
    assert step(dk=96) == 4 and step(dv=100) == 4 and step(dv=0) == 4 and step(dv=8192) == 4
    assert step(s_in=ODD) == 2 and step(s_out=ODD) == 2
    assert step(rows=-1) == 1 and step(slots=0) == 1
    assert step(index=None, rows=5) == 1          # a slot for each row without an index
    assert step(s_out=ctypes.c_void_p(0x10100)) == 1   # overlaps state_in
    assert b"overlap" in _lib.lib().qfn_last_error()
    assert step(rows=0) == 0 and step(rows=0, q=None, out=None) == 0


def chunk(q=FAKE, cu=FAKE, n=2, T=100, s_in=FAKE, s_out=FAR, ws=FAR, bytes_=None, H=4, Hk=2, dk=128, dv=128):
    L = _lib.lib()
    if bytes_ is None:
        bytes_ = L.qfn_deltanet_chunk_workspace(T, n, H, Hk, dk, dv)
    return L.qfn_deltanet_chunk(q, FAKE, FAKE, FAKE, FAKE, STRIDES, cu, n, T, s_in, s_out, FAKE, H, Hk, dk, dv, ws,
                                bytes_, None)


def test_chunk_refusals():
    assert chunk(q=None) == 1 and chunk(s_out=None) == 1
    assert chunk(n=-1) == 1 and chunk(T=-1) == 1 and chunk(n=0, cu=None) == 1
    assert chunk(cu=None, n=3) == 1               # 100 tokens are not three equal sequences
    assert chunk(Hk=3) == 1 and chunk(dk=32) == 4 and chunk(dv=48) == 4
    assert chunk(s_in=ODD) == 2
    assert chunk(s_out=ctypes.c_void_p(0x10100)) == 1
    assert chunk(T=2 ** 31) == 4
    need = _lib.lib().qfn_deltanet_chunk_workspace(100, 2, 4, 2, 128, 128)
    assert need > 0 and chunk(bytes_=need - 1) == 5 and chunk(ws=None) == 5
    assert chunk(ws=ctypes.c_void_p(0x7f0000000010)) == 2
    assert _lib.lib().qfn_deltanet_chunk_workspace(100, 0, 4, 2, 128, 128) == 0
    assert chunk(n=0) == 0 and chunk(n=0, T=0) == 0 and chunk(n=0, T=0, q=None, s_out=None) == 0


def test_gated_norm_refusals():
    def f(x=FAKE, w=FAKE, wd=0, rows=4, heads=2, dim=128):
        return _lib.lib().qfn_gated_norm(x, 256, 128, FAKE, 256, 128, w, wd, FAKE, rows, heads, dim, 1e-6, None)
    assert f(x=None) == 1 and f(w=None) == 1 and f(wd=2) == 1
    assert f(rows=-1) == 1 and f(heads=0) == 1 and f(dim=0) == 1
    assert f(rows=0, x=None) == 0


def test_norm_residual_refusals():
    def f(block=FAKE, bd=1, gate=None, kind=0, nxt=None, normed=None, rows=4, dim=128):
        return _lib.lib().qfn_norm_residual(block, bd, 128, FAKE, 1, 128, None, 1, gate, kind, 1, 1, 1, 1.0, nxt, 1, FAKE,
                                            normed, rows, dim, 1e-6, None)
    assert f(block=None) == 1 and f(bd=3) == 1 and f(kind=3) == 1 and f(kind=-1) == 1
    assert f(kind=1) == 1 and f(nxt=FAKE) == 1    # a kind without a gate, a weight without an output
    assert f(rows=-1) == 1 and f(dim=0) == 1 and f(dim=32769) == 4
    assert f(rows=0) == 0


def test_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    bf, B, T, H, d = torch.bfloat16, 2, 3, 2, 64
    q, v, g, b = (torch.zeros(B, T, H, d, dtype=bf), torch.zeros(B, T, H, d, dtype=bf), torch.zeros(B, T, H),
                  torch.zeros(B, T, H, dtype=bf))
    S = torch.zeros(B, H, d, d)
    with pytest.raises(ValueError, match="CUDA"):
        deltanet.chunk_gated_delta_rule(q, q, v, g, b)
    with pytest.raises(ValueError, match="heads, dk"):
        deltanet.chunk_gated_delta_rule(q[0], q[0], v[0], g[0], b[0])
    with pytest.raises(ValueError, match="cu_seqlens takes one"):
        deltanet.chunk_gated_delta_rule(q, q, v, g, b, cu_seqlens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="value must be"):
        deltanet.chunk_gated_delta_rule(q, q, v[:, :2], g, b)
    with pytest.raises(ValueError, match="beta must be"):
        deltanet.chunk_gated_delta_rule(q, q, v, g, b[..., None])
    with pytest.raises(ValueError, match="out must be"):
        deltanet.chunk_gated_delta_rule(q, q, v, g, b, out=v[:, :, :1])
    with pytest.raises(ValueError, match="CUDA"):
        deltanet.step_gated_delta_rule(q[0], q[0], v[0], g[0], b[0], S)
    with pytest.raises(ValueError, match="CUDA"):
        norms.gated_rms_norm(q, q, torch.ones(d))
    with pytest.raises(ValueError, match="same shape"):
        norms.gated_rms_norm(q, q[0], torch.ones(d))
    with pytest.raises(ValueError, match="CUDA"):
        norms.norm_residual(q[0, 0], q[0, 0])


@pytest.mark.gpu
def test_wrappers_refuse_wrong_types_and_shapes_on_the_device():
    bf, T, H, d, dev = torch.bfloat16, 3, 2, 64, "cuda"
    q, v, g, b = (torch.zeros(T, H, d, dtype=bf, device=dev), torch.zeros(T, H, d, dtype=bf, device=dev),
                  torch.zeros(T, H, device=dev), torch.zeros(T, H, dtype=bf, device=dev))
    S, ix = torch.zeros(T, H, d, d, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)

    def step(q=q, k=q, v=v, g=g, b=b, S=S, **kw):
        return deltanet.step_gated_delta_rule(q, k, v, g, b, S, **kw)

    for kw in (dict(q=q.float()), dict(v=v.half()), dict(g=g.double()), dict(b=b.float()), dict(S=S.half()),
               dict(state_index=ix.long()), dict(out=torch.zeros(T, H, d, device=dev))):
        with pytest.raises(TypeError):
            step(**kw)
    for kw in (dict(k=q[:2]), dict(v=v[:, :1]), dict(g=g[:2]), dict(b=b[:, :1]), dict(S=S[:, :1]), dict(S=S[:2]),
               dict(S=S.transpose(2, 3)), dict(state_index=ix[:2]), dict(out_state=S[:2]), dict(out=v[:2]),
               dict(out=v), dict(g=g.cpu()), dict(state_index=ix.cpu())):
        with pytest.raises(ValueError):
            step(**kw)
    for bad in (dict(q=q[..., :32], k=q[..., :32], S=S[:, :, :32].contiguous()),
                dict(v=v[..., :40].contiguous(), S=S[..., :40].contiguous())):
        with pytest.raises(RuntimeError, match="unsupported"):
            step(**bad)
    both = torch.zeros(2 * T - 1, H, d, d, device=dev)
    with pytest.raises(RuntimeError, match="overlap"):
        step(S=both[:T], out_state=both[T - 1:])

    def chunk(cu=None, S0=None, S1=None, out=None):
        return deltanet.chunk_gated_delta_rule(q[None], q[None], v[None], g[None], b[None], S0, cu, S1, out)

    with pytest.raises(TypeError):
        chunk(cu=torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(TypeError):
        chunk(S0=S[:1].double())
    for kw in (dict(cu=torch.zeros(2, dtype=torch.int32)), dict(cu=torch.zeros(0, dtype=torch.int32, device=dev)),
               dict(S0=S), dict(S1=S[:2]), dict(out=v), dict(out=v[None])):
        with pytest.raises(ValueError):
            chunk(**kw)
    w = torch.ones(d, device=dev)
    with pytest.raises(TypeError):
        norms.gated_rms_norm(q.float(), q, w)
    with pytest.raises(TypeError):
        norms.gated_rms_norm(q, q, w.half())
    with pytest.raises(ValueError):
        norms.gated_rms_norm(q, q, w[:32])
    x = torch.zeros(T, d, dtype=bf, device=dev)
    with pytest.raises(TypeError):
        norms.norm_residual(x.half(), x)
    for kw in (dict(post_weight=w[:3]), dict(gate=x[:2]), dict(gate=x[:, :3]), dict(next_weight=w.cpu()),
               dict(out=x[:2])):
        with pytest.raises(ValueError):
            norms.norm_residual(x, x.clone(), **kw)
    with pytest.raises(TypeError):
        norms.norm_residual(x, x, out=x.float())
