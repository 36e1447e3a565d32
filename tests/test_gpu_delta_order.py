"""Calls that follow one another on one state, nothing between them: each reads what the one before wrote."""
import pytest
import torch

import deltanet
import synthetic
from test_gpu_delta_batch import check, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_steps_on_one_state_in_a_graph():
    """40 one-token steps captured one behind the other, against 40 single calls."""
    T, H, Hk, d = 40, 32, 16, 128
    q, k, v, g, beta, S0 = (t.to(DEV) for t in synthetic.deltanet_inputs(T, H, Hk, d, d, 3))
    args = [[x[t][None, None].contiguous() for x in (q, k, v, g, beta)] for t in range(T)]
    one = S0[None].clone()
    want = []
    for a in args:
        want.append(deltanet.recurrent_gated_delta_rule(*a, one)[0])
        torch.cuda.synchronize()
    S = S0[None].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [deltanet.recurrent_gated_delta_rule(*a, S)[0] for a in args]
    for _ in range(5):
        S.copy_(S0[None])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(S, one) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n", [4, 70])
def test_prompt_then_steps_in_a_graph(n):
    """A prompt of n tokens, a one-token step of either kind, and again, all in place on one state."""
    T, H, Hk, d = 2 * n + 4, 8, 4, 128
    q, k, v, g, beta, S0 = (t.to(DEV) for t in synthetic.deltanet_inputs(T, H, Hk, d, d, 4))
    x = (q, k, v, g, beta)
    S = S0[None].clone()

    def run():
        outs, t = [], 0
        for _ in range(2):
            outs.append(deltanet.chunk_gated_delta_rule(*(a[t:t + n][None] for a in x), S, final_state=S)[0][0])
            t += n
            outs.append(deltanet.recurrent_gated_delta_rule(*(a[t][None, None] for a in x), S)[0][0])
            outs.append(deltanet.step_gated_delta_rule(*(a[t + 1][None] for a in x), S)[0])
            t += 2
        return torch.cat(outs)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    ref = oracle(*x, S0)
    first = None
    for _ in range(5):
        S.copy_(S0[None])
        graph.replay()
        torch.cuda.synchronize()
        check(out, S[0], ref, T)
        first = first if first is not None else (out.clone(), S.clone())
        assert torch.equal(out, first[0]) and torch.equal(S, first[1])
