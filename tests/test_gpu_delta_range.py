"""The gated delta rule over prompts where magnitudes differ: between the columns of a head, between the
tokens of a chunk, around a cleared state, with decays above one, and where a value is not finite.

Tolerances, for each column and token.  u = 2^-24 is half a step of fp32.  `top` is the column's largest
magnitude so far, |S| and |v|, decayed as the state is; a column depends on no other one, so neither does its
tolerance:

    tol_state = u (16 + 4 sqrt(tokens)) top

An output is formed from bf16 terms before its rounding: S^T q from two terms of S (2^-16 of each product),
P d from two terms of either factor (2^-16 each, and 2^-16 for the product of the two low ones); 2^-14 of the sum
of the products' magnitudes `mag` covers them, and half a bf16 step the rounding.  Below 2^-126 bf16 has steps of
2^-133, so that the last term of S, P and d is off by up to 2^-134 however small the value is.  What that adds is below
FLOOR = 2^-126, the smallest normal number of both types: to a state 64 tokens' 2^-134 |k|, |k| <= 4 an element of
these inputs, = 2^-126; to an output 2^-134 sum|q| <= 2^-134 from S (|q| = dk^-1/2), 64 dk^-1/2 2^-134 <= 2^-131 from d,
as much from P where |d| <= 1.
"""
import math

import pytest
import torch

import _lib
import deltanet
import synthetic
from test_gpu_delta_segments import walks

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
FLOOR = 2.0 ** -126


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert _lib.device_status() == 0


def inputs(T, H, Hk, dk, dv, seed):
    q, k, v, g, beta, _ = synthetic.deltanet_inputs(T, H, Hk, dk, dv, seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    S0 = torch.randn(H, dk, dv, device=DEV, generator=gen) * 0.05
    return [t.to(DEV) for t in (q, k, v, g, beta)] + [S0]


def recurrence(q, k, v, g, beta, S):
    """Token by token in 64 bits -> out, S, mag, top, each token's [T, H, dv]; S the last."""
    H, r = v.shape[1], v.shape[1] // q.shape[1]
    q, k = (t.double().repeat_interleave(r, 1) for t in (q, k))
    q = q / ((q * q).sum(-1, keepdim=True) + 1e-6).sqrt() / q.shape[-1] ** 0.5
    k = k / ((k * k).sum(-1, keepdim=True) + 1e-6).sqrt()
    v, g, beta, S = v.double(), g.double(), beta.double(), S.double()
    M, top = S.abs(), S.abs().amax(1)
    out, mag, tops = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(v)
    for t in range(v.shape[0]):
        a = g[t].exp()[:, None, None]
        S, M, top = S * a, M * a, top * a[:, 0]
        d = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * d[:, None]
        M = M + k[t].abs()[:, :, None] * d.abs()[:, None]
        top = torch.maximum(torch.maximum(top, S.abs().amax(1)), v[t].abs())
        out[t] = torch.einsum("hkv,hk->hv", S, q[t])
        mag[t] = torch.einsum("hkv,hk->hv", M, q[t].abs())
        tops[t] = top
    return out, S, mag, tops


def half_step(x):
    """Half a bf16 step at |x| (the smallest normal number's below it)."""
    e = torch.frexp(x.abs().clamp_min(2.0 ** -126))[1]
    return torch.ldexp(torch.ones_like(x), e - 9)


def close(out, S, ref, tokens=None):
    r_out, r_S, mag, top = ref
    T = r_out.shape[0]
    n = slice(0, T if tokens is None else tokens)
    tol = U * (16 + 4 * math.sqrt(T)) * top
    err = (out[n].double() - r_out[n]).abs()
    lim = half_step(r_out[n]) + 2.0 ** -14 * mag[n] + 2 * tol[n] + FLOOR
    assert (err <= lim).all(), f"out: {(err / lim).max():.2f} x tolerance"
    if S is not None:
        err, lim = (S.double() - r_S).abs(), tol[-1][:, None] + FLOOR
        assert (err <= lim).all(), f"state: {(err / lim).max():.2f} x tolerance"


def chunk(many, q, k, v, g, beta, S0):
    """One sequence (the walk of few states), or as the last of 32 (the walk of many: 128 states, a block of 128
    columns each)."""
    N = 32 if many else 1
    rep = [t.repeat(N, *[1] * (t.dim() - 1)).unflatten(0, (N, t.shape[0])) for t in (q, k, v, g, beta)]
    out, S = deltanet.chunk_gated_delta_rule(*rep, S0.repeat(N, 1, 1, 1))
    return out[N - 1], S[N - 1]


def arrange(case, q, k, v, g, beta, S0):
    T, dv = v.shape[0], v.shape[-1]
    if case == "columns":       # neighbouring columns of one state, 2^60 apart
        s = torch.tensor([0, -12, -20, -40, 20], device=DEV)[torch.arange(dv, device=DEV) % 5]
        v, S0 = torch.ldexp(v.float(), s).to(v.dtype), torch.ldexp(S0, s)
    elif case == "token":       # one token far above the others: those before it keep their digits
        v[T // 4] *= 2.0 ** 24
    elif case == "carried":     # a large carried state that decays within the chunk
        S0 = S0 * 2.0 ** 24
        g[:] = -1.0
    elif case == "cleared":     # a large carried state, cleared in the first chunk
        S0 = S0 * 2.0 ** 30
        g[20] = -float("inf")
    elif case == "cleared-late":
        v[:70] *= 2.0 ** 30
        g[75] = -float("inf")
        g[77] = -1e30
    elif case == "rise":        # the state grows by e^60 at one token
        g[30] = 60.0
    elif case == "rising":
        g = 0.1 * g.abs()
    elif case == "beta":        # steps past the projection
        beta = (1 + beta.float()).to(beta.dtype)
    elif case == "one-product":   # outputs of one product each: nothing averages the operands' roundings
        v[1:] = 0
        S0 = S0 * (torch.arange(S0.shape[1], device=DEV) == 7)[:, None]
        q[:, :, :7] = 0
        q[:, :, 8:] = 0
    return q, k, v, g, beta, S0


CASES = ["columns", "token", "carried", "cleared", "cleared-late", "rise", "rising", "beta", "one-product"]


SHAPES = [(128, 128), (64, 96), (64, 128)]   # those of the tests below


@pytest.mark.parametrize("dk,dv", SHAPES)
@pytest.mark.parametrize("many", [False, True])
def test_the_walk_is_the_one_meant(many, dk, dv):
    names, _ = walks(lambda: chunk(many, *inputs(150, 4, 2, dk, dv, seed=41)))
    assert names <= {"walk_warp" if many else "walk_quad"}


@pytest.mark.parametrize("dk,dv", SHAPES[:2])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_magnitudes(case, many, dk, dv):
    args = arrange(case, *inputs(150, 4, 2, dk, dv, seed=41))
    out, S = chunk(many, *args)
    close(out, S, recurrence(*args))


@pytest.mark.parametrize("case", CASES)
def test_magnitudes_token_by_token(case):
    """dk = 256 and short calls run the recurrence: the same values, the same tolerances."""
    args = arrange(case, *inputs(90, 2, 1, 256, 32, seed=41))
    out, S = chunk(False, *args)
    close(out, S, recurrence(*args))


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("what", ["g-nan", "g-inf", "beta-nan", "beta-inf", "q-nan", "k-nan", "k-inf", "v-nan", "v-inf", "overflow"])
@pytest.mark.parametrize("at", [6, 40, 100])
def test_not_finite_from_its_token_on(what, at, many, dk):
    """One head's decay, beta, query, key or value that is not finite, or products that overflow, leave its earlier
    tokens and the other heads alone."""
    T, H = 150, 4
    q, k, v, g, beta, S0 = inputs(T, H, H, dk, 128, seed=7)
    clean = recurrence(q, k, v, g, beta, S0)
    if what == "overflow":      # every step multiplies what the head holds along its key by -40
        k[at:at + 40, 1] = k[at, 1]
        beta[at:at + 40, 1] = 41
    elif what[0] in "qkv":
        {"q": q, "k": k, "v": v}[what[0]][at, 1, 3] = float(what.split("-")[1])
    else:
        (g if what[0] == "g" else beta)[at, 1] = float(what.split("-")[1])
    out, S = chunk(many, q, k, v, g, beta, S0)
    close(out, None, clean, tokens=at)
    heads = [0, 2, 3]
    close(out[:, heads], S[heads], (clean[0][:, heads], clean[1][heads], clean[2][:, heads], clean[3][:, heads]))
    if what == "q-nan":         # the state has no part in it
        assert out[at, 1].isnan().all()
        close(torch.where(out.isnan(), clean[0].to(out.dtype), out), S, clean)
    elif what[0] == "v":        # nor have the other columns
        keep = torch.ones(H, 128, dtype=torch.bool, device=DEV)
        keep[1, 3] = False
        assert not out[at:, 1, 3].isfinite().any() and not S[1, :, 3].isfinite().any()
        close(torch.where(keep, out, clean[0].to(out.dtype)), torch.where(keep[:, None], S, clean[1].float()), clean)
    else:
        assert not out[-1, 1].isfinite().any() and not S[1].isfinite().all(0).any()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bad", ["inf", "nan"])
@pytest.mark.parametrize("at", [1, 5, 64, 127])
def test_decay_not_finite_leaves_the_token_before(at, bad, many):
    T, H = 150, 4
    q, k, v, g, beta, S0 = inputs(T, H, H, 64, 128, seed=8)
    clean = recurrence(q, k, v, g, beta, S0)
    g[at, 2] = float(bad)
    out, S = chunk(many, q, k, v, g, beta, S0)
    close(out, None, clean, tokens=at)
    heads = [0, 1, 3]
    close(out[:, heads], S[heads], (clean[0][:, heads], clean[1][heads], clean[2][:, heads], clean[3][:, heads]))
    assert not out[at:, 2].isfinite().any() and not S[2].isfinite().any()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_not_finite_carried_column(bad, many):
    T, H = 100, 4
    q, k, v, g, beta, S0 = inputs(T, H, 2, 64, 128, seed=9)
    clean = recurrence(q, k, v, g, beta, S0)
    S0 = S0.clone()
    S0[1, 3, 5] = float(bad)
    S0[2, :, 120] = float(bad)
    out, S = chunk(many, q, k, v, g, beta, S0)
    keep = torch.ones(H, 128, dtype=torch.bool, device=DEV)
    keep[1, 5] = keep[2, 120] = False
    assert not out.isfinite()[:, ~keep].any() and not S.isfinite()[1, :, 5].any() and not S.isfinite()[2, :, 120].any()
    close(torch.where(keep, out, clean[0].to(out.dtype)), torch.where(keep[:, None], S, clean[1].float()), clean)
