"""Outputs of the batched delta rule and the norms that share memory with something that is still read are refused."""
import ctypes

import pytest
import torch

import _lib
import deltanet
import norms

P = ctypes.c_void_p
IN, STATE, STATE2, OUT, WS = 0x10000, 0x7f0000000000, 0x7f1000000000, 0x7f2000000000, 0x7f3000000000
STRIDES = (ctypes.c_int64 * 10)(*([128] * 10))
STATE_BYTES = 4 * 4 * 128 * 128   # one slot of 4 heads of 128 x 128
ROW_BYTES = 2 * 4 * 128           # one row of out


def last_error():
    return _lib.lib().qfn_last_error()


def step(out, s_in=STATE, s_out=STATE2):
    return _lib.lib().qfn_deltanet_step_batch(P(IN), P(IN), P(IN), P(IN), P(IN), STRIDES, P(IN), 3, P(s_in), P(s_out), P(out),
                                              2, 4, 2, 128, 128, None)


def chunk(out, s_in=STATE, s_out=STATE2, T=100):
    L = _lib.lib()
    return L.qfn_deltanet_chunk(P(IN), P(IN), P(IN), P(IN), P(IN), STRIDES, P(IN), 3, T, P(s_in), P(s_out), P(out), 4, 2, 128,
                                128, P(WS), L.qfn_deltanet_chunk_workspace(T, 3, 4, 2, 128, 128), None)


@pytest.mark.parametrize("state", [STATE, STATE2])
def test_out_over_a_state_is_refused_by_the_library(state):
    for f, rows in ((step, 2), (chunk, 100)):
        for out in (state, state + STATE_BYTES, state + 3 * STATE_BYTES - 16, state - rows * ROW_BYTES + 16):
            assert f(out) == 1 and b"out overlaps a state" in last_error(), hex(out)
    assert chunk(state, T=4) == 1 and b"out overlaps a state" in last_error()   # the token recurrence
    assert step(STATE, s_out=STATE) == 1 and b"out overlaps a state" in last_error()   # in place


@pytest.mark.skipif(torch.cuda.is_available(), reason="neighbours would be launched")
def test_neighbours_pass_the_check():
    for f, rows in ((step, 2), (chunk, 100)):
        for out in (OUT, STATE + 3 * STATE_BYTES, STATE2 - rows * ROW_BYTES):
            assert f(out) not in (0, 1, 2, 5)   # no device here: past the checks of arguments


bf, dev = torch.bfloat16, "cuda"


def at(buf, offset, dtype, *shape):
    """A tensor of `shape` at byte `offset` of buf."""
    n = torch.empty(shape, dtype=dtype, device="meta").nbytes
    return buf[offset:offset + n].view(dtype).view(shape)


def rows(T, H=2, d=64):
    return [torch.zeros(T, H, d, dtype=bf, device=dev) for _ in range(3)] + [torch.zeros(T, H, device=dev),
                                                                            torch.zeros(T, H, dtype=bf, device=dev)]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 20])
def test_chunk_refuses_shared_memory(T):
    H, d = 2, 64
    S_shape, o_shape = (1, H, d, d), (1, T, H, d)
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)

    def call(q, k, v, g, b, **kw):
        return deltanet.chunk_gated_delta_rule(*(t[None] for t in (q, k, v, g, b)), **kw)

    x = rows(T)
    S, out = at(buf, 0, torch.float32, *S_shape), at(buf, 16, bf, *o_shape)
    with pytest.raises(RuntimeError, match="out overlaps a state"):
        call(*x, initial_state=S, out=out)
    with pytest.raises(RuntimeError, match="out overlaps a state"):
        call(*x, final_state=S, out=out)
    with pytest.raises(ValueError, match="out overlaps cu_seqlens"):
        c = at(buf, 64, torch.int32, 2)
        c.copy_(cu)
        call(*x, out=out, cu_seqlens=c)
    with pytest.raises(ValueError, match="final_state overlaps cu_seqlens"):
        call(*x, final_state=S, cu_seqlens=c)
    for i, (name, dtype) in enumerate((("query", bf), ("key", bf), ("value", bf), ("g", torch.float32), ("beta", bf))):
        y = list(x)
        y[i] = at(buf, 4096, dtype, *x[i].shape)
        with pytest.raises(ValueError, match=f"final_state overlaps {name}"):
            call(*y, final_state=S)
        with pytest.raises(ValueError, match=f"out overlaps {name}"):
            call(*y, out=at(buf, 4096, bf, *o_shape))
    call(*x, initial_state=S, final_state=S, out=at(buf, S.nbytes, bf, *o_shape), cu_seqlens=cu)   # neighbours


@pytest.mark.gpu
def test_step_refuses_shared_memory():
    T, H, d = 3, 2, 64
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    x = rows(T)
    S = at(buf, 0, torch.float32, T, H, d, d)
    with pytest.raises(RuntimeError, match="out overlaps a state"):
        deltanet.step_gated_delta_rule(*x, S, out=at(buf, S.nbytes - 16, bf, T, H, d))
    with pytest.raises(RuntimeError, match="out overlaps a state"):
        deltanet.step_gated_delta_rule(*x, S, out_state=torch.empty_like(S), out=at(buf, 0, bf, T, H, d))
    ix = at(buf, 32, torch.int32, T)
    with pytest.raises(ValueError, match="out_state overlaps state_index"):
        deltanet.step_gated_delta_rule(*x, S, state_index=ix)
    with pytest.raises(ValueError, match="out overlaps state_index"):
        deltanet.step_gated_delta_rule(*x, torch.zeros_like(S), state_index=ix, out=at(buf, 0, bf, T, H, d))
    for i, (name, dtype) in enumerate((("query", bf), ("key", bf), ("value", bf), ("g", torch.float32), ("beta", bf))):
        y = list(x)
        y[i] = at(buf, 4096, dtype, *x[i].shape)
        with pytest.raises(ValueError, match=f"out_state overlaps {name}"):
            deltanet.step_gated_delta_rule(*y, S)
    deltanet.step_gated_delta_rule(*x, S, out=at(buf, S.nbytes, bf, T, H, d))


@pytest.mark.gpu
def test_norm_residual_refuses_shared_memory():
    T, D = 3, 64
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device=dev)
    x, w, out = torch.zeros(T, D, dtype=bf, device=dev), at(buf, 64, bf, D), at(buf, 0, bf, T, D)
    for kw in (dict(post_weight=w), dict(next_weight=w), dict(gate=at(buf, 64, bf, T, 1)), dict(gate=at(buf, 64, bf, T, D))):
        with pytest.raises(ValueError, match=f"out overlaps {next(iter(kw))}"):
            norms.norm_residual(x, x.clone(), out=out, **kw)
    with pytest.raises(ValueError, match="out overlaps block"):
        norms.norm_residual(at(buf, 64, bf, T, D), x, out=out)
    norms.norm_residual(x, out, post_weight=at(buf, out.nbytes, bf, D), out=out)
