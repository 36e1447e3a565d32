"""The chunked delta rule where its work is divided: over segments of the workspace, between the two walks, and in
the walk of many states over blocks of 128 and of 64 columns.  Each test makes sure that its call is divided so.

Heads are independent, so a few of them are compared with the token recurrence in 64 bits; tolerances as in
test_gpu_delta_batch.py (a state u (16 + 4 sqrt(tokens)) of the head's largest value, an output a rounding to bf16 and
2^-10 of its products' magnitudes).
"""
import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import _lib
import deltanet
from test_gpu_delta_batch import check, no_wait_ran_out, offsets, oracle   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(T, H, Hk, dk, dv, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    return [rnd(T, Hk, dk).to(torch.bfloat16), rnd(T, Hk, dk).to(torch.bfloat16), rnd(T, H, dv).to(torch.bfloat16),
            -rnd(T, H).abs() * 0.3, torch.sigmoid(rnd(T, H)).to(torch.bfloat16)]


def walks(call):
    """The walks that a call launches, and its result.  A profiler may miss a kernel, so it may take another call; where
    there is no profiler the set stays empty."""
    for _ in range(5):
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA], acc_events=True) as prof:
            got = call()
            torch.cuda.synchronize()
        names = {n for e in prof.events() for n in ("walk_quad", "walk_warp") if f"dn_{n}_kernel" in e.name}
        if names:
            break
    return names, got


def segment_slots(n_seqs, H, Hk, dk, dv):
    """Slots that a segment of the workspace holds: sequence n starts at slot cu[n] // 64 + n."""
    f = _lib.lib().qfn_deltanet_chunk_workspace
    slot = f(64 * 50, n_seqs, H, Hk, dk, dv) - f(64 * 49, n_seqs, H, Hk, dk, dv)
    return f(2 ** 30, n_seqs, H, Hk, dk, dv) // slot


def compare(heads, x, S0, cu, out, S):
    q, k, v, g, beta = x
    r = v.shape[1] // q.shape[1]
    keys = [h // r for h in heads]
    for n in range(len(cu) - 1):
        at = slice(int(cu[n]), int(cu[n + 1]))
        ref = oracle(q[at][:, keys], k[at][:, keys], v[at][:, heads], g[at][:, heads], beta[at][:, heads],
                     None if S0 is None else S0[n, heads])
        check(out[at][:, heads], S[n, heads], ref, at.stop - at.start)


@pytest.mark.parametrize("more", [0, 1, 64, 4600], ids=["ends-on-an-edge", "one-token-past", "a-chunk-past", "third-segment"])
def test_one_sequence_over_segments(more):
    H, dk, dv = 32, 128, 32
    fit = segment_slots(1, H, H, dk, dv)
    T = fit * 64 + more
    x = inputs(T, H, H, dk, dv, seed=3)
    S0 = torch.randn(1, H, dk, dv, device=DEV) * 0.05
    names, (out, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S0))
    segments = -(-(T // 64 + 1) // fit)
    assert segments == (3 if more > 4000 else 2) and names <= {"walk_quad"}
    compare([0, 17], x, S0, [0, T], out[0], S)
    carried = S0.clone()   # in place: later segments read what earlier ones wrote
    out2, _ = deltanet.chunk_gated_delta_rule(*(t[None] for t in x), carried, final_state=carried)
    assert torch.equal(out2, out) and torch.equal(carried, S)


def ragged(kind, fit):
    return {"crosses": [100, fit * 64 + 70, 0, 30],             # the second sequence crosses the edge
            "ends-on-the-edge": [fit * 64, 5, 200],             # its last chunk is the segment's last slot
            "empty-on-the-edge": [fit * 64 - 64, 0, 300, 0],    # an empty one has the next segment's first slot
            "starts-on-the-edge": [fit * 64 - 64, 130, 64],     # so has one with tokens
            "two-edges": [10, 2 * fit * 64 + 1, 63]}[kind]


@pytest.mark.parametrize("walk,dv", [("walk_quad", 32), ("walk_warp", 128)])
@pytest.mark.parametrize("kind", ["crosses", "ends-on-the-edge", "empty-on-the-edge", "starts-on-the-edge", "two-edges"])
def test_ragged_batch_over_segments(kind, walk, dv):
    H, dk = 128, 128
    fit = segment_slots(3, H, H, dk, dv)
    lens = ragged(kind, fit)
    cu = offsets(lens)
    x = inputs(sum(lens), H, H, dk, dv, seed=4)
    S0 = torch.randn(len(lens), H, dk, dv, device=DEV) * 0.05
    names, (out, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S0, cu))
    segments = -(-(sum(lens) // 64 + len(lens)) // fit)
    assert segments == (3 if kind == "two-edges" else 2) and names <= {walk}
    assert out.isfinite().all() and S.isfinite().all()
    compare([1, 127], x, S0, cu.tolist(), out[0], S)
    carried = S0.clone()
    out2, _ = deltanet.chunk_gated_delta_rule(*(t[None] for t in x), carried, cu, carried)
    assert torch.equal(out2, out) and torch.equal(carried, S)


@pytest.mark.parametrize("walk,dv", [("walk_quad", 32), ("walk_warp", 128)])
def test_bad_bounds_over_segments(walk, dv):
    H, dk = 128, 128
    fit = segment_slots(3, H, H, dk, dv)
    T = fit * 64 + 300
    x = inputs(T, H, H, dk, dv, seed=5)
    out = torch.full((1, T, H, dv), 7.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, T - 100, T - 200, T], dtype=torch.int32, device=DEV)
    names, (_, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), cu_seqlens=cu, out=out))
    assert names <= {walk} and (out == 7).all() and S.isnan().all()


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dv", [32, 96, 128, 160, 192])
@pytest.mark.parametrize("kind", ["equal", "short", "long"])
def test_walk_of_many_states(kind, dv, dk):
    """Blocks of 128 columns, the last partly filled, and ("long") of 64 columns for sequences past their share."""
    H, Hk, N = 8, 4, 16 if dv == 96 else 24   # 128 states of 96 columns fill one round of blocks of 128
    lens = {"equal": [90] * N, "short": [70, 0, 1, 64] * (N // 4), "long": [0] * (N - 4) + [600, 3, 1000, 5]}[kind]
    cu = offsets(lens)
    x = inputs(sum(lens), H, Hk, dk, dv, seed=6)
    S0 = torch.randn(len(lens), H, dk, dv, device=DEV) * 0.05
    names, (out, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S0, cu))
    assert names <= {"walk_quad" if dv == 32 else "walk_warp"}
    compare(list(range(H)), x, S0, cu.tolist(), out[0], S)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dv", [32, 96, 128, 160])
def test_walk_of_few_states(dv, dk):
    lens, H, Hk = [130, 64, 1, 0, 65], 4, 2
    cu = offsets(lens)
    x = inputs(sum(lens), H, Hk, dk, dv, seed=7)
    S0 = torch.randn(len(lens), H, dk, dv, device=DEV) * 0.05
    names, (out, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S0, cu))
    assert names <= {"walk_quad"}
    compare(list(range(H)), x, S0, cu.tolist(), out[0], S)


@pytest.mark.parametrize("many", [False, True])
def test_rows_past_32_bits(many):
    """Token rows 2^20 elements apart: the last ones lie past 2^31 elements."""
    T, H, Hk, dk, dv, N = 2400, 4, 2, 128, 128, 32 if many else 1
    x = inputs(T, H, Hk, dk, dv, seed=8)
    S0 = torch.randn(N, H, dk, dv, device=DEV) * 0.05
    cu = offsets([T // N] * N)
    want, S_want = deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S0, cu)
    row = torch.empty(T, 2 ** 20, dtype=torch.bfloat16, device=DEV)
    assert (T - 1) * 2 ** 20 > 2 ** 31
    far, at = [], 0
    for t in x[:3]:
        far.append(row[:, at:at + t[0].numel()].view(t.shape))
        far[-1].copy_(t)
        at += t[0].numel()
    names, (out, S) = walks(lambda: deltanet.chunk_gated_delta_rule(*(t[None] for t in far + x[3:]), S0, cu))
    assert names <= {"walk_warp" if many else "walk_quad"} and torch.equal(out, want) and torch.equal(S, S_want)


def test_states_past_32_bits():
    H, dk, dv, N = 32, 128, 128, 2 ** 31 // (32 * 128 * 128) + 3
    lens = [0] * (N - 2) + [70, 9]
    cu = offsets(lens)
    x = inputs(sum(lens), H, H, dk, dv, seed=9)
    S = torch.zeros(N, H, dk, dv, device=DEV)
    S[-2:] = torch.randn(2, H, dk, dv, device=DEV) * 0.05
    first = S[-2:].clone()
    out, got = deltanet.chunk_gated_delta_rule(*(t[None] for t in x), S, cu, S)
    assert got is S and not S[:-2].any()
    compare([0, 31], x, first, [0, 70, 79], out[0], S[-2:])
