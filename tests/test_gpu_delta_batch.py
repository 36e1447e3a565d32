"""GPU parity of the batched gated delta rule (deltanet.chunk_gated_delta_rule,
deltanet.step_gated_delta_rule) against the token recurrence in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32.  A state element passes through
a few fp32 roundings per token and through sums over dk (16 u covers one
token: the norms' reciprocal roots, the products and the partial sums of a
dot product); the tokens' errors are independent, so they add like
sqrt(tokens):

    tol_state = u (16 + 4 sqrt(tokens)) max|S|       (max over the head, with S0 and v)

An output is rounded once to bf16 (2^-8 of its value) and, where chunks of tokens are
multiplied on the tensor cores, formed from f16 factors: two roundings of
2^-11 on each product of a chunk, one on each product with the state, 2^-10 in
all of the sum of the products' magnitudes `mag`, which the oracle carries
along (M = exp(g) M + |k| |d|^T, mag = M^T |q|).
"""
import math

import pytest
import torch

import _lib
import deltanet
import fp8gemv
import norms
import synthetic

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert _lib.device_status() == 0


def inputs(tokens, H, Hk, dk, dv, seed, strided=True):
    """q, k, v as views of one row per token (as a projection leaves them) or dense; g, beta."""
    q, k, v, g, beta, _ = synthetic.deltanet_inputs(max(tokens, 1), H, Hk, dk, dv, seed)
    q, k, v, g, beta = (t[:tokens].to(DEV) for t in (q, k, v, g, beta))
    if strided:
        row = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
        q, k, v = (t.view(tokens, -1, d) for t, d in zip(row.split([Hk * dk, Hk * dk, H * dv], 1), (dk, dk, dv)))
    return q, k, v, g, beta


def states(n, H, dk, dv, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return torch.randn(n, H, dk, dv, device=DEV, generator=gen) * 0.05


def oracle(q, k, v, g, beta, S):
    """The token recurrence of one sequence in 64 bits -> out, S, mag, scale of S for each head."""
    H, r = v.shape[1], v.shape[1] // q.shape[1]
    q, k = (t.double().repeat_interleave(r, 1) for t in (q, k))
    q = q / ((q * q).sum(-1, keepdim=True) + 1e-6).sqrt() / q.shape[-1] ** 0.5
    k = k / ((k * k).sum(-1, keepdim=True) + 1e-6).sqrt()
    v, g, beta = v.double(), g.double(), beta.double()
    S = torch.zeros(H, q.shape[-1], v.shape[-1], dtype=torch.float64, device=DEV) if S is None else S.double()
    M, top = S.abs(), S.abs().amax((1, 2))
    out, mag = torch.zeros_like(v), torch.zeros_like(v)
    for t in range(v.shape[0]):
        a = g[t].exp()[:, None, None]
        S, M = torch.where(a == 0, 0.0, S) * a, torch.where(a == 0, 0.0, M) * a
        d = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * d[:, None]
        M = M + k[t].abs()[:, :, None] * d.abs()[:, None]
        out[t] = torch.einsum("hkv,hk->hv", S, q[t])
        mag[t] = torch.einsum("hkv,hk->hv", M, q[t].abs())
    top = torch.maximum(torch.maximum(top, S.abs().amax((1, 2))), v.abs().amax((0, 2)) if v.shape[0] else top)
    return out, S, mag, top


def check(out, S, ref, tokens):
    r_out, r_S, mag, top = ref
    tol = (U * (16 + 4 * math.sqrt(max(tokens, 1))) * top)[:, None]
    err = (S.double() - r_S).abs()
    assert (err <= tol[:, :, None]).all(), f"state: {(err / tol[:, :, None]).max():.2f} x tolerance"
    err, tol = (out.double() - r_out).abs(), 2.0 ** -8 * r_out.abs() + 2.0 ** -10 * mag + 2 * tol
    assert (err <= tol).all(), f"out: {(err / tol).max():.2f} x tolerance" if err.numel() else ""


def offsets(lens, start=0):
    cu = [start]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def run_ragged(lens, H, Hk, dk, dv, seed, carried, **kw):
    cu = offsets(lens)
    T = int(cu[-1])
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed, **kw)
    S0 = states(len(lens), H, dk, dv, seed) if carried else None
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0, cu)
    assert out.shape == (1, T, H, dv) and out.dtype == torch.bfloat16 and S.dtype == torch.float32
    for n, length in enumerate(lens):
        at = slice(int(cu[n]), int(cu[n + 1]))
        check(out[0, at], S[n], oracle(q[at], k[at], v[at], g[at], beta[at], S0[n] if carried else None), length)


HEADS = [(4, 2, 128, 128), (2, 2, 64, 96), (3, 1, 128, 32), (2, 1, 256, 64), (1, 1, 64, 160)]


@pytest.mark.parametrize("H,Hk,dk,dv", HEADS)
@pytest.mark.parametrize("lens", [[1], [15], [64], [65], [130], [0, 1, 63, 64, 65, 0, 200, 16, 0]], ids=str)
def test_chunk_matches_recurrence(lens, H, Hk, dk, dv):
    run_ragged(lens, H, Hk, dk, dv, seed=sum(lens) + dk, carried=len(lens) > 1)


@pytest.mark.parametrize("carried", [False, True])
def test_chunk_long_sequence(carried):
    run_ragged([2049], 2, 1, 128, 128, seed=5, carried=carried)


def test_chunk_more_than_one_segment():
    """More chunks than one workspace holds: the state goes from segment to segment through memory."""
    run_ragged([100, 6000, 0, 40], 32, 32, 128, 32, seed=8, carried=True)


@pytest.mark.parametrize("lens,H,Hk,dk,dv", [
    ([70, 1, 0, 64, 129, 65, 200, 33, 16, 128, 5, 63], 8, 4, 128, 128),
    ([90] * 20, 8, 8, 64, 96),
    ([90] * 50, 4, 2, 128, 64),
    ([65, 0, 100] * 10, 8, 2, 64, 160),
    ([20] * 70 + [100], 3, 1, 128, 128)], ids=lambda x: str(x)[:20])
def test_chunk_many_states(lens, H, Hk, dk, dv):
    """Enough states for the walk of many sequences (blocks of 128 columns, the last of them partly filled)."""
    run_ragged(lens, H, Hk, dk, dv, seed=len(lens) + dv, carried=True)


def test_chunk_few_and_many_states_agree():
    """The two walks on the same sequences: one alone, and as one of many."""
    H, Hk, dk, dv, T, N = 4, 2, 128, 128, 200, 40
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed=12, strided=False)
    S0 = states(1, H, dk, dv, 3)
    one, S_one = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0)
    rep = [t.repeat(N, *[1] * (t.dim() - 1)).unflatten(0, (N, T)) for t in (q, k, v, g, beta)]
    many, S_many = deltanet.chunk_gated_delta_rule(*rep, S0.repeat(N, 1, 1, 1))
    assert (many == many[:1]).all() and (S_many == S_many[:1]).all()
    ref = oracle(q, k, v, g, beta, S0[0])
    check(one[0], S_one[0], ref, T)
    check(many[N - 1], S_many[N - 1], ref, T)


@pytest.mark.parametrize("case", ["reset", "strong", "none", "zero-keys", "beta0", "same-keys", "large", "small"])
def test_chunk_extremes_many_states(case):
    """The cases of test_chunk_extremes in the walk of many sequences."""
    H, Hk, dk, dv, T, N = 4, 1, 128, 128, 150, 40
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed=22, strided=False)
    S0 = states(1, H, dk, dv, 8)
    q, k, v, g, beta, S0 = extreme(case, q, k, v, g, beta, S0)
    rep = [t.repeat(N, *[1] * (t.dim() - 1)).unflatten(0, (N, T)) for t in (q, k, v, g, beta)]
    out, S = deltanet.chunk_gated_delta_rule(*rep, S0.repeat(N, 1, 1, 1))
    check(out[N - 1], S[N - 1], oracle(q, k, v, g, beta, S0[0]), T)


def test_chunk_nan_stays_in_its_column_many_states():
    H, dk, dv, T, N = 4, 64, 128, 150, 40
    q, k, v, g, beta = inputs(T, H, 1, dk, dv, seed=4, strided=False)
    v[T // 2, 1, 40] = float("nan")
    v[T // 2, 1, 9] = float("inf")
    rep = [t.repeat(N, *[1] * (t.dim() - 1)).unflatten(0, (N, T)) for t in (q, k, v, g, beta)]
    out, S = deltanet.chunk_gated_delta_rule(*rep)
    keep = torch.ones(H, dv, dtype=torch.bool, device=DEV)
    keep[1, [9, 40]] = False
    assert not out[0, T // 2:].isfinite()[:, ~keep].any() and out[0, :T // 2].isfinite().all()
    assert not S[0].isfinite()[1][:, [9, 40]].any()
    vv = torch.where(v.isfinite(), v, 0)
    r_out, r_S, mag, top = oracle(q, k, vv, g, beta, None)
    zero = lambda t, m: torch.where(m, t.double(), 0.0)
    check(zero(out[3], keep), zero(S[3], keep[:, None]), (zero(r_out, keep), zero(r_S, keep[:, None]), mag, top), T)


def test_chunk_bad_bounds_many_states():
    T, N, H, dk, dv = 400, 40, 4, 64, 128
    q, k, v, g, beta = inputs(T, H, 1, dk, dv, seed=2)
    out = torch.full((1, T, H, dv), 7.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.arange(N + 1, dtype=torch.int32, device=DEV) * 10
    cu[17] = 400
    _, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], out=out, cu_seqlens=cu)
    assert (out == 7).all() and S.isnan().all()


def test_chunk_many_short_sequences():
    gen = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 9, (150,), generator=gen).tolist()
    run_ragged(lens, 2, 2, 64, 32, seed=11, carried=True)


@pytest.mark.parametrize("lens", [[3], [40, 41]])
def test_chunk_strides_and_alignment(lens):
    """Dense tensors, views that start off a 16-byte boundary, transposed heads, copies of a strided last dimension."""
    H, Hk, dk, dv = 2, 1, 64, 64
    T = sum(lens)
    cu = offsets(lens)
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed=3, strided=False)
    S0 = states(len(lens), H, dk, dv, 4)
    want, S_want = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0, cu)

    def odd(t):   # the same values one element off the allocation's start, rows of an odd stride
        flat = torch.empty(T, t[0].numel() + 3, dtype=t.dtype, device=DEV)
        flat[:, 1:1 + t[0].numel()] = t.flatten(1)
        return flat[:, 1:1 + t[0].numel()].view(t.shape) if t[0].numel() else t

    def headmajor(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def lastmajor(t):
        return t.transpose(0, -1).contiguous().transpose(0, -1)

    for f in (odd, headmajor, lastmajor):
        out, S = deltanet.chunk_gated_delta_rule(f(q)[None], f(k)[None], f(v)[None], f(g)[None], f(beta)[None], S0, cu)
        assert torch.equal(out, want) and torch.equal(S, S_want), f.__name__


@pytest.mark.parametrize("T", [5, 100])
def test_chunk_equal_batch_and_pieces(T):
    """B rows without cu_seqlens; the same tokens in two pieces with the state handed on, the second
    in place; a token step after them."""
    B, H, Hk, dk, dv = 3, 2, 1, 128, 64
    q, k, v, g, beta = (t.unflatten(0, (B, T + 1)) for t in inputs(B * (T + 1), H, Hk, dk, dv, seed=T))
    S0 = states(B, H, dk, dv, 1)
    kept = S0.clone()
    args = [t[:, :T] for t in (q, k, v, g, beta)]
    out, S = deltanet.chunk_gated_delta_rule(*args, S0)
    assert torch.equal(S0, kept)
    cut = T // 3
    out1, mid = deltanet.chunk_gated_delta_rule(*(t[:, :cut] for t in args), S0)
    out2, S2 = deltanet.chunk_gated_delta_rule(*(t[:, cut:] for t in args), mid, final_state=mid)
    assert S2.data_ptr() == mid.data_ptr()
    last, S3 = deltanet.step_gated_delta_rule(*(t[:, T] for t in (q, k, v, g, beta)), S)
    assert S3 is S
    for b in range(B):
        ref = oracle(*(t[b] for t in args), S0[b])
        check(torch.cat([out1, out2], 1)[b], S2[b], ref, T)
        check(out[b], S2[b], ref, T)
        ref = oracle(*(t[b] for t in (q, k, v, g, beta)), S0[b])
        check(last[b][None], S[b], tuple(x[-1:] if i in (0, 2) else x for i, x in enumerate(ref)), T + 1)


@pytest.mark.parametrize("H,Hk,dk,dv", HEADS)
@pytest.mark.parametrize("N,T", [(3, 8), (20, 1), (20, 8), (20, 9)])
def test_chunk_batch_of_short_sequences(N, T, H, Hk, dk, dv):
    """Equal lengths on both sides of the token recurrence's longest; the bounds given as well."""
    q, k, v, g, beta = (t.unflatten(0, (N, T)) for t in inputs(N * T, H, Hk, dk, dv, 31))
    S0 = states(N, H, dk, dv, 31)
    out, S = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, S0)
    flat = [t.flatten(0, 1)[None] for t in (q, k, v, g, beta)]
    out_cu, S_cu = deltanet.chunk_gated_delta_rule(*flat, S0, offsets([T] * N))
    for n in range(N):
        ref = oracle(q[n], k[n], v[n], g[n], beta[n], S0[n])
        check(out[n], S[n], ref, T)
        check(out_cu[0, n * T:(n + 1) * T], S_cu[n], ref, T)
    carried = S0.clone()
    deltanet.chunk_gated_delta_rule(q, k, v, g, beta, carried, final_state=carried)
    assert torch.equal(carried, S)


@pytest.mark.parametrize("T", [12, 90])
def test_chunk_leaves_rows_outside_the_sequences(T):
    """(Padded tokens before, between the last sequence and the end.)"""
    H, Hk, dk, dv = 2, 2, 64, 32
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed=2)
    for t in (q, k, v, g, beta):   # nothing outside may be read either
        t[:3] = float("nan")
        t[T - 2:] = float("nan")
    cu = offsets([4, T - 9], start=3)
    out = torch.full((1, T, H, dv), 7.0, dtype=torch.bfloat16, device=DEV)
    got, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], cu_seqlens=cu, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[0, :3] == 7).all() and (out[0, T - 2:] == 7).all()
    for n, (a, b) in enumerate([(3, 7), (7, T - 2)]):
        check(out[0, a:b], S[n], oracle(q[a:b], k[a:b], v[a:b], g[a:b], beta[a:b], None), b - a)


@pytest.mark.parametrize("cu", [[0, 50, 40, 90], [-1, 10, 20, 30], [0, 10, 20, 91], [0, 2 ** 31 - 1, 5, 90], [90, 0, 0, 0]])
def test_chunk_bad_bounds(cu):
    T, H, dk, dv = 90, 2, 64, 32
    q, k, v, g, beta = inputs(T, H, 1, dk, dv, seed=2)
    out = torch.full((1, T, H, dv), 7.0, dtype=torch.bfloat16, device=DEV)
    _, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], out=out,
                                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert (out == 7).all() and S.isnan().all()


def test_chunk_nothing_to_do():
    H, dk, dv = 2, 64, 32
    q, k, v, g, beta = (t[:0] for t in inputs(1, H, 1, dk, dv, seed=2))
    S0 = states(2, H, dk, dv, 1)
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0, offsets([0, 0]))
    assert out.shape == (1, 0, H, dv) and torch.equal(S, S0)
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], cu_seqlens=offsets([]))
    assert S.shape == (0, H, dk, dv)
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None])
    assert S.shape == (1, H, dk, dv) and (S == 0).all()
    q, k, v, g, beta = inputs(70, H, 1, dk, dv, seed=2)   # rows of which no sequence is left
    out = torch.full((1, 70, H, dv), 7.0, dtype=torch.bfloat16, device=DEV)
    _, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], cu_seqlens=offsets([]), out=out)
    assert S.shape == (0, H, dk, dv) and (out == 7).all()
    _, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0, offsets([0, 0]), out=out)
    assert torch.equal(S, S0) and (out == 7).all()


def extreme(case, q, k, v, g, beta, S0):
    T = q.shape[0]
    if case == "reset":
        g[T // 2] = -float("inf")
        g[T // 2 + 2] = -1e30
    elif case == "strong":
        g = g - 60 * (torch.arange(T, device=DEV) % 3 == 0)[:, None]
    elif case == "none":
        g = torch.zeros_like(g)
    elif case == "zero-keys":
        k[::2] = 0
        q[1::3] = 0
    elif case == "beta0":
        beta = torch.zeros_like(beta)
    elif case == "same-keys":
        k[:] = k[0]
        beta = torch.ones_like(beta)
    elif case == "large":
        v, S0 = v * 2.0 ** 60, S0 * 2.0 ** 60
        k, q = k * 2.0 ** 40, q * 2.0 ** -3
    elif case == "small":
        v, S0 = v * 2.0 ** -60, S0 * 2.0 ** -60
        k, q = k * 2.0 ** -8, q * 2.0 ** 50
    return q, k, v, g, beta, S0


@pytest.mark.parametrize("T", [9, 150])
@pytest.mark.parametrize("case", ["reset", "strong", "none", "zero-keys", "beta0", "same-keys", "large", "small"])
def test_chunk_extremes(case, T):
    """A decay of zero in mid-sequence, strong and no decay, keys and betas of zero, one key
    repeated, values far from one."""
    H, Hk, dk, dv = 2, 1, 128, 32
    q, k, v, g, beta = inputs(T, H, Hk, dk, dv, seed=21, strided=False)
    S0 = states(1, H, dk, dv, 8)
    q, k, v, g, beta, S0 = extreme(case, q, k, v, g, beta, S0)
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], S0,
                                             torch.tensor([0, T], dtype=torch.int32, device=DEV))
    check(out[0], S[0], oracle(q, k, v, g, beta, S0[0]), T)


@pytest.mark.parametrize("T", [9, 150])
def test_chunk_nan_stays_in_its_sequence_and_column(T):
    H, dk, dv = 2, 64, 64
    q, k, v, g, beta = inputs(2 * T, H, 1, dk, dv, seed=4, strided=False)
    v[T // 2, 1, 40] = float("nan")
    v[T // 2, 1, 9] = float("inf")
    out, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], cu_seqlens=offsets([T, T]))
    bad = torch.zeros(H, dv, dtype=torch.bool, device=DEV)
    bad[1, [9, 40]] = True
    assert not S[0].isfinite()[:, :, :][1][:, [9, 40]].any() and not out[0, T // 2:T].isfinite()[:, bad].any()
    assert out[0, :T // 2].isfinite().all() and out[0, T:].isfinite().all() and S[1].isfinite().all()
    vv = torch.where(v.isfinite(), v, 0)
    ref = oracle(q[:T], k[:T], vv[:T], g[:T], beta[:T], None)
    keep = ~bad
    r_out, r_S, mag, top = ref
    zero = lambda t, m: torch.where(m, t.double(), 0.0)
    check(zero(out[0, :T], keep), zero(S[0], keep[:, None]), (zero(r_out, keep), zero(r_S, keep[:, None]), mag, top), T)


@pytest.mark.parametrize("n_seqs", [1, 40])
@pytest.mark.parametrize("at", [3, 20, 40, 55, 70])
def test_chunk_nan_key_leaves_earlier_tokens(at, n_seqs):
    """A key that is not a number spoils its head from its token on, never the tokens before it."""
    H, Hk, dk, dv, T = 4, 4, 128, 128, 130
    q, k, v, g, beta = (t.unflatten(0, (n_seqs, T)) for t in inputs(n_seqs * T, H, Hk, dk, dv, 17))
    k = k.clone()
    k[0, at, 1, 5] = float("nan")
    out, S = deltanet.chunk_gated_delta_rule(q, k, v, g, beta)
    assert out[0, at:, 1].isnan().all() and S[0, 1].isnan().all()
    ref_out, _, mag, top = oracle(*(t[0, :at] for t in (q, k, v, g, beta)), None)
    tol = 2.0 ** -8 * ref_out.abs() + 2.0 ** -10 * mag + 2 * (U * (16 + 4 * math.sqrt(T)) * top)[:, None]
    assert ((out[0, :at].double() - ref_out).abs() <= tol).all()
    others = [0, 2, 3]
    ref = oracle(*(t[0][:, others] for t in (q, k, v, g, beta)), None)
    check(out[0][:, others], S[0, others], ref, T)


def test_chunk_repeats_bit_for_bit_on_another_stream_and_in_a_graph():
    lens, H, Hk, dk, dv = [70, 3, 129], 4, 2, 128, 64
    stream_and_graph(lens, H, Hk, dk, dv, (lens, [1, 200, 1], [0, 0, 202]))


def test_chunk_many_states_on_another_stream_and_in_a_graph():
    lens = [30] * 40
    stream_and_graph(lens, 4, 2, 64, 128, (lens, [1200] + [0] * 39, [29] * 39 + [69]))


def stream_and_graph(lens, H, Hk, dk, dv, replays):
    cu = offsets(lens)
    q, k, v, g, beta = (t[None] for t in inputs(sum(lens), H, Hk, dk, dv, seed=6))
    S0 = states(len(lens), H, dk, dv, 2)
    out, S = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, S0, cu)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):   # two calls at once
        for s in (a, b):
            with torch.cuda.stream(s):
                got.append(deltanet.chunk_gated_delta_rule(q, k, v, g, beta, S0, cu))
    torch.cuda.synchronize()
    for o, s in got:
        assert torch.equal(o, out) and torch.equal(s, S)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o1, s1 = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, S0, cu)
        o2, s2 = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, s1, cu)
    # other lengths at replay: the bounds are read on the device
    for lens2 in replays:
        cu.copy_(offsets(lens2))
        graph.replay()
        e1, f1 = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, S0, cu)
        e2, f2 = deltanet.chunk_gated_delta_rule(q, k, v, g, beta, f1, cu)
        assert all(torch.equal(x, y) for x, y in ((o1, e1), (s1, f1), (o2, e2), (s2, f2)))


# ------------------------------------------------------------------ one token of each request
@pytest.mark.parametrize("H,Hk,dk,dv", HEADS + [(32, 16, 128, 128)])
@pytest.mark.parametrize("rows", [1, 5, 33])
def test_step_matches_recurrence(rows, H, Hk, dk, dv):
    q, k, v, g, beta = inputs(rows, H, Hk, dk, dv, seed=rows + dk)
    pool = states(rows + 3, H, dk, dv, 3)
    index = torch.randperm(rows + 3, generator=torch.Generator().manual_seed(1))[:rows].to(torch.int32).to(DEV)
    if rows > 2:
        index[1] = -1
        index[rows - 1] = -7
    kept, new = pool.clone(), torch.full_like(pool, 5.0)
    out, S = deltanet.step_gated_delta_rule(q, k, v, g, beta, pool, index, out_state=new)
    assert S is new and torch.equal(pool, kept)
    out2, S2 = deltanet.step_gated_delta_rule(q, k, v, g, beta, pool, index)
    assert S2 is pool and torch.equal(out, out2)
    named = index[index >= 0].long()
    rest = torch.ones(rows + 3, dtype=torch.bool, device=DEV)
    rest[named] = False
    assert (new[rest] == 5).all() and torch.equal(pool[rest], kept[rest]) and torch.equal(pool[named], new[named])
    for r in range(rows):
        if index[r] < 0:
            assert (out[r] == 0).all()
            continue
        ref = oracle(*(t[r:r + 1] for t in (q, k, v, g, beta)), kept[index[r].long()])
        check(out[r:r + 1], pool[index[r].long()], ref, 1)


def test_step_is_the_one_token_rule():
    """Row for row the existing one-token entry point's values, up to fp32 summation order."""
    H, Hk, dk, dv, R = 8, 4, 128, 128, 4
    q, k, v, g, beta = inputs(R, H, Hk, dk, dv, seed=1, strided=False)
    pool = states(R, H, dk, dv, 2)
    one = pool.clone()
    out, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, pool)
    for r in range(R):
        o, _ = deltanet.recurrent_gated_delta_rule(*(t[r][None, None] for t in (q, k, v, g, beta)), one[r:r + 1])
        assert (o[0, 0].float() - out[r].float()).abs().max() <= 2.0 ** -7 * out[r].float().abs().max()
    assert (one - pool).abs().max() <= 40 * U * one.abs().max()


def test_step_wrong_slots():
    """A slot named twice, and slots past the pool: NaN for those rows, no state touched by them."""
    R, H, dk, dv = 6, 2, 64, 32
    q, k, v, g, beta = inputs(R, H, 1, dk, dv, seed=1)
    pool = states(4, H, dk, dv, 2)
    kept = pool.clone()
    index = torch.tensor([2, 0, 2, 4, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    out, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, pool, index)
    assert out[[2, 3, 4]].isnan().all() and (out[5] == 0).all()
    assert torch.equal(pool[[1, 3]], kept[[1, 3]])
    for r in (0, 1):
        check(out[r:r + 1], pool[int(index[r])], oracle(*(t[r:r + 1] for t in (q, k, v, g, beta)), kept[int(index[r])]), 1)


def test_step_reset_and_large_pool():
    """exp(-inf) clears a state; slots whose offset passes 32 bits."""
    H, dk, dv = 32, 128, 128
    slots = 2 ** 31 // (H * dk * dv) + 2
    pool = torch.empty(slots, H, dk, dv, device=DEV)
    q, k, v, g, beta = inputs(2, H, H, dk, dv, seed=1)
    index = torch.tensor([slots - 1, 0], dtype=torch.int32, device=DEV)
    S0 = states(2, H, dk, dv, 2)
    pool[index.long()] = S0
    g[1] = -float("inf")
    out, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, pool, index)
    for r in range(2):
        check(out[r:r + 1], pool[int(index[r])], oracle(*(t[r:r + 1] for t in (q, k, v, g, beta)), S0[r]), 1)


def test_step_captured_with_padding_at_replay():
    R, H, dk, dv = 8, 4, 128, 64
    q, k, v, g, beta = inputs(R, H, 2, dk, dv, seed=7)
    pool = states(R, H, dk, dv, 2)
    index = torch.arange(R, dtype=torch.int32, device=DEV)
    deltanet.step_gated_delta_rule(q, k, v, g, beta, pool.clone(), index)
    work = pool.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, work, index)
        out2, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, work, index)
    for live in (R, 3):
        index.copy_(torch.arange(R) - R * (torch.arange(R) >= live))
        work.copy_(pool)
        graph.replay()
        mine = pool.clone()
        e1, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, mine, index)
        e2, _ = deltanet.step_gated_delta_rule(q, k, v, g, beta, mine, index)
        assert torch.equal(out, e1) and torch.equal(out2, e2) and torch.equal(work, mine)
        assert (out[live:] == 0).all()


# ------------------------------------------------------------------ the layer they make up
@pytest.mark.parametrize("lens", [[1, 1, 1], [33, 70]])
def test_layer_between_quantized_products(lens):
    """linear(q|k|v) and linear(z) -> chunk -> gated norm -> linear(out) -> norm and residual, then one decoded
    token of each request through the same layer, against the same chain in 64 bits from each stage's input."""
    H, Hk, dk, dv, hid = 4, 2, 64, 64, 256
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)

    def rnd(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    def fp8(n, k):
        w = rnd(n, k) * k ** -0.5
        s = w.abs().amax(1) / 448
        return (w / s[:, None]).to(torch.float8_e4m3fn), s

    w_qkv, w_z, w_o = fp8((2 * Hk * dk + H * dv), hid), fp8(H * dv, hid), fp8(hid, H * dv)
    w_norm, w_post, w_next = 1 + 0.1 * rnd(dv), 1 + 0.1 * rnd(hid), 1 + 0.1 * rnd(hid)
    T, N = sum(lens), len(lens)
    x, residual = rnd(T + N, hid).to(torch.bfloat16), rnd(T + N, hid).to(torch.bfloat16)
    g, beta = -rnd(T + N, H).abs(), torch.sigmoid(rnd(T + N, H)).to(torch.bfloat16)
    cu = offsets(lens)

    def layer(rows, S, step):
        n = rows.stop - rows.start
        qkv, z = fp8gemv.linear(x[rows], *w_qkv), fp8gemv.linear(x[rows], *w_z)
        q, k, v = (t.view(n, -1, d) for t, d in zip(qkv.split([Hk * dk, Hk * dk, H * dv], 1), (dk, dk, dv)))
        if step:
            o, S = deltanet.step_gated_delta_rule(q, k, v, g[rows], beta[rows], S)
        else:
            o, S = deltanet.chunk_gated_delta_rule(q[None], k[None], v[None], g[rows][None], beta[rows][None], S, cu)
            o = o[0]
        y = norms.gated_rms_norm(o, z.view(n, H, dv), w_norm)
        block = fp8gemv.linear(y.view(n, H * dv), *w_o)
        r, nx = norms.norm_residual(block, residual[rows], w_post, next_weight=w_next, scale=0.5)
        return q, k, v, o, S, z, y, block, r, nx

    q, k, v, o, S, z, y, block, r, nx = layer(slice(0, T), None, False)
    before = S.clone()
    for n in range(N):
        at = slice(int(cu[n]), int(cu[n + 1]))
        check(o[at], S[n], oracle(q[at], k[at], v[at], g[at], beta[at], None), lens[n])
    q2, k2, v2, o2, S2, z2, y2, block2, r2, nx2 = layer(slice(T, T + N), S, True)
    assert S2 is S
    for n in range(N):
        check(o2[n:n + 1], S[n], oracle(q2[n:n + 1], k2[n:n + 1], v2[n:n + 1], g[T + n:T + n + 1],
                                        beta[T + n:T + n + 1], before[n]), 1)
    for o_, z_, y_, block_, r_, nx_, rows in ((o, z, y, block, r, nx, slice(0, T)), (o2, z2, y2, block2, r2, nx2, slice(T, T + N))):
        od, zd = o_.double(), z_.double().view(o_.shape)
        want = od / (od.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w_norm.double() * zd * torch.sigmoid(zd)
        assert ((y_.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want.abs()).all()
        bd = block_.double()
        want = residual[rows].double() + 0.5 * bd / (bd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w_post.double()
        assert ((r_.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all()
        want = want / (want.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w_next.double()
        assert ((nx_.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all()
