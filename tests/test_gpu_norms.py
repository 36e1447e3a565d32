"""GPU parity of norms.gated_rms_norm and norms.norm_residual against the formulas in 64 bits.

Tolerances: one rounding of the output (2^-8 of the value for bf16, 2^-24 for fp32) and fp32
arithmetic before it.  The sum of squares of a row adds in at most 64 steps on one thread
and ten of a tree, the rest (root, reciprocal, sigmoid, products) is a dozen roundings:
ARITH = 2^-24 * 96 < 2^-17 relative to the magnitudes that are added.
"""
import pytest
import torch

import norms

pytestmark = pytest.mark.gpu
DEV = "cuda"
ARITH = 2.0 ** -17
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rnd(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=gen) * scale).to(dtype)


def rms(x, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def near(got, want, mag=None):
    mag = want.abs() if mag is None else mag
    tol = HALF_STEP[got.dtype] * want.abs() + ARITH * mag + 2.0 ** -126   # below it fp32 and bf16 have no normal numbers
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"{(err / tol).max():.2f} x tolerance"


def gated_ref(x, z, w, eps):
    z = z.double()
    return rms(x, eps) * w.double() * z * torch.sigmoid(z)


@pytest.mark.parametrize("D", [1, 7, 8, 64, 96, 100, 128, 136, 256, 264, 1000])
@pytest.mark.parametrize("T,H", [(1, 1), (5, 3), (70, 4)])
def test_gated_norm(T, H, D):
    x, z = rnd(T, H, D, seed=1), rnd(T, H, D, seed=2, scale=3)
    for wd in (torch.float32, torch.bfloat16):
        w = rnd(D, seed=3, dtype=wd)
        y = norms.gated_rms_norm(x, z, w)
        assert y.shape == x.shape and y.dtype == torch.bfloat16
        near(y, gated_ref(x, z, w, 1e-6))


def test_gated_norm_views_and_shapes():
    T, H, D = 9, 4, 64
    w = rnd(D, seed=3)
    buf = rnd(T, 2 * H * D + 8, seed=5)
    x, z = buf[:, :H * D].view(T, H, D), buf[:, H * D + 8:].view(T, H, D)
    want = norms.gated_rms_norm(x.contiguous(), z.contiguous(), w)
    near(want, gated_ref(x, z, w, 1e-6))
    odd = rnd(T, H * D + 3, seed=5)
    odd[:, 1:H * D + 1] = x.reshape(T, -1)
    for a, b in ((x, z), (odd[:, 1:H * D + 1].view(T, H, D), z), (x.transpose(0, 1).contiguous().transpose(0, 1), z),
                 (x.transpose(0, 2).contiguous().transpose(0, 2), z.clone())):
        got = norms.gated_rms_norm(a, b, w)
        near(got, gated_ref(x, z, w, 1e-6))
    assert torch.equal(norms.gated_rms_norm(x[None], z[None], w)[0], want)
    near(norms.gated_rms_norm(x[:, 0], z[:, 0], w), gated_ref(x[:, 0], z[:, 0], w, 1e-6))
    assert norms.gated_rms_norm(x[:0], z[:0], w).shape == (0, H, D)


def test_gated_norm_extremes():
    x, z, w = rnd(6, 1, 128, seed=1), rnd(6, 1, 128, seed=2), torch.ones(128, device=DEV)
    x[0] = 0
    z[1] = -200
    z[2] = 200
    x[3] *= 2.0 ** -40
    x[4] *= 2.0 ** 40
    x[5, 0, 3] = float("nan")
    y = norms.gated_rms_norm(x, z, w, eps=1e-5)
    near(y[:5], gated_ref(x[:5], z[:5], w, 1e-5))
    assert y[5].isnan().all()


def residual_ref(block, residual, post, gate, scale, nxt, eps, sigmoid):
    p = block.double() if post is None else rms(block, eps) * post.double()
    if gate is not None:
        gate = gate.double() if gate.dim() == 2 else gate.double()[:, None]
        p = p * (torch.sigmoid(gate) if sigmoid else gate)
    r = residual.double() + scale * p
    mag = residual.double().abs() + abs(scale) * p.abs()
    if nxt is None:
        return r, mag, None, None
    # an error of ARITH * mag in r moves n by that over the row's root, and through the row's mean by
    # less than the row's mean error
    root = (r.square().mean(-1, keepdim=True) + eps).sqrt()
    n_mag = (mag + r.abs() / root * mag.square().mean(-1, keepdim=True).sqrt() + r.abs()) / root * nxt.double().abs()
    return r, mag, r / root * nxt.double(), n_mag


def run(T, D, bd, rd, gate_shape, post, nxt, seed=0, sigmoid=True, wd=torch.bfloat16, gd=torch.bfloat16, scale=0.7):
    block, residual = rnd(T, D, seed=seed + 1, dtype=bd), rnd(T, D, seed=seed + 2, dtype=rd, scale=2)
    gate = None if gate_shape is None else rnd(*gate_shape, seed=seed + 3, dtype=gd, scale=2)
    w_post = rnd(D, seed=seed + 4, dtype=wd) if post else None
    w_next = rnd(D, seed=seed + 5, dtype=wd) if nxt else None
    r, n = norms.norm_residual(block, residual, w_post, gate, scale, w_next, sigmoid=sigmoid)
    assert r.dtype == rd and r.shape == (T, D)
    want, mag, n_want, n_mag = residual_ref(block, residual, w_post, gate, scale, w_next, 1e-6, sigmoid)
    near(r, want, mag)
    if nxt:
        assert n.dtype == torch.bfloat16
        near(n, n_want, n_mag)
    else:
        assert n is None


@pytest.mark.parametrize("D", [1, 3, 8, 255, 256, 2557, 2560, 4104, 8192, 9001, 16384, 32760, 32767])
@pytest.mark.parametrize("T", [1, 7])
def test_norm_residual_sizes(T, D):
    run(T, D, torch.bfloat16, torch.bfloat16, (T, D), True, True)


@pytest.mark.parametrize("bd", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rd", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate,sigmoid", [(None, True), ("row", True), ("row1", False), ("all", True), ("all", False)])
@pytest.mark.parametrize("post,nxt", [(True, True), (True, False), (False, True), (False, False)])
def test_norm_residual_kinds(bd, rd, gate, sigmoid, post, nxt):
    T, D = 5, 512
    shape = {None: None, "row": (T,), "row1": (T, 1), "all": (T, D)}[gate]
    for D_, wd, gd in ((D, torch.bfloat16, torch.float32), (D, torch.float32, torch.bfloat16)):
        run(T, D_, bd, rd, shape, post, nxt, sigmoid=sigmoid, wd=wd, gd=gd, scale=-1.5)


def test_norm_residual_views_in_place_and_empty():
    T, D = 6, 320
    buf = rnd(T, 3 * D + 1, seed=1)
    w = rnd(D, seed=2)
    for block, residual, gate in ((buf[:, :D], buf[:, D:2 * D], buf[:, 2 * D:3 * D]),
                                  (buf[:, 1:D + 1], buf[:, D:2 * D], buf[:, 3 * D:]),
                                  (buf[:, :D], rnd(D, T, seed=3).t(), None)):
        r, n = norms.norm_residual(block, residual, w, gate, next_weight=w)
        want, mag, n_want, n_mag = residual_ref(block, residual, w, gate, 1.0, w, 1e-6, True)
        near(r, want, mag)
        near(n, n_want, n_mag)
    block, residual = buf[:, :D].contiguous(), buf[:, D:2 * D].contiguous()
    r, n = norms.norm_residual(block, residual, w, next_weight=w)
    mine = residual.clone()
    r2, n2 = norms.norm_residual(block, mine, w, next_weight=w, out=mine)
    assert r2.data_ptr() == mine.data_ptr() and torch.equal(mine, r) and torch.equal(n2, n)
    with pytest.raises(ValueError, match="overlaps"):
        norms.norm_residual(block, residual, w, out=block)
    big = torch.empty(T + 1, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        norms.norm_residual(block, big[:T], w, out=big[1:])
    r, n = norms.norm_residual(block[:0], residual[:0], w, next_weight=w)
    assert r.shape == n.shape == (0, D)


def test_norm_residual_extremes():
    T, D = 5, 2560
    block, residual = rnd(T, D, seed=1, dtype=torch.float32), rnd(T, D, seed=2)
    w = torch.ones(D, device=DEV)
    block[0] = 0
    block[1] *= 2.0 ** 50
    residual[2] = 0
    block[2] = 0
    residual[3] *= 2.0 ** 50
    block[4, 7] = float("nan")
    r, n = norms.norm_residual(block, residual, w, next_weight=w)
    want, mag, n_want, n_mag = residual_ref(block, residual, w, None, 1.0, w, 1e-6, True)
    near(r[:4], want[:4], mag[:4])
    near(n[:4], n_want[:4], n_mag[:4])
    assert r[4].isnan().all() and n[4].isnan().all()


def test_norms_in_a_graph_and_on_another_stream():
    T, H, D = 40, 4, 64
    x, z, w, res, wr = rnd(T, H, D, seed=1), rnd(T, H, D, seed=2), rnd(D, seed=3), rnd(T, H * D, seed=4), rnd(H * D, seed=5)

    def both():
        y = norms.gated_rms_norm(x, z, w)
        return (y,) + norms.norm_residual(y.view(T, H * D), res, wr, next_weight=wr)

    want = both()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    x.mul_(-0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, both()))
