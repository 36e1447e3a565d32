"""Gated delta rule of the DeltaNet (linear-attention) layers on B200.

recurrent_gated_delta_rule (libqfn's qfn_deltanet_step) is a drop-in for
qwen_engine.recurrent_gated_delta_rule at T == 1 (qwen_engine.py:158-174), the
call QwenEngine.deltanet makes for every linear-attention layer of every
decoded token (qwen_engine.py:718-719).

chunk_gated_delta_rule (qfn_deltanet_chunk) runs the same rule over prompts:
sequences of any length, ragged batches of them, with a state carried in and
out.  step_gated_delta_rule (qfn_deltanet_step_batch) runs one token for each
request of a batch, with the requests' states in slots of a pool.

Per token and value head (value head h uses key head h // (H // Hq)):

    q = l2norm(q) / sqrt(dk);  k = l2norm(k)       l2norm: x * rsqrt(sum x^2 + 1e-6)
    S = exp(g) * S;  d = beta * (v - S^T k);  S = S + k d^T;  out = bf16(S^T q)

The states and every sum are fp32.  The prompts' chunks multiply on the tensor
cores: what the state is made of is taken with fp32's 24 bits, what only reaches
the bf16 outputs with 16 of them, each value with an exponent of its own.  -inf
in g clears a finite state.  g is a decay, g <= 0; growth is taken too, as long as
it stays below e^88 within 64 tokens.  q and k rows have norms below 2^63; where
both are below 2^-50 their products lose digits.

All three are forward only; the batched two refuse a tensor that requires a
gradient while gradients are recorded.
"""
import torch

from _lib import check, lib, on_device, op, require_cuda, stream_of


def recurrent_gated_delta_rule(query, key, value, g, beta, initial_state):
    """query, key [1, 1, Hq, dk] bf16 (Hq = H, the engine's repeated heads, or the
    H / r key heads) . value [1, 1, H, dv] bf16 . g [1, 1, H] fp32 . beta [1, 1, H]
    bf16 . initial_state [1, H, dk, dv] fp32 -> (out [1, 1, H, dv] bf16, S).

    S is initial_state updated in place (the engine stores the returned state,
    st["S"] = S, so the in-place update is what it keeps)."""
    for name, t, dt in (("query", query, torch.bfloat16), ("key", key, torch.bfloat16),
                        ("value", value, torch.bfloat16), ("beta", beta, torch.bfloat16),
                        ("g", g, torch.float32), ("initial_state", initial_state, torch.float32)):
        require_cuda(name, t, dt)
    if query.dim() != 4 or query.shape[0] != 1 or query.shape[1] != 1:
        raise ValueError(f"query must be [1, 1, heads, dk] (one token), got {tuple(query.shape)}")
    Hq, dk = query.shape[2], query.shape[3]
    H, dv = value.shape[2], value.shape[3]
    if tuple(key.shape) != tuple(query.shape) or value.shape[:2] != (1, 1) or H % Hq:
        raise ValueError("key must match query; value [1, 1, H, dv] with H a multiple of query's heads")
    if g.numel() != H or beta.numel() != H or tuple(initial_state.shape) != (1, H, dk, dv):
        raise ValueError(f"g, beta [1, 1, {H}] and initial_state [1, {H}, {dk}, {dv}] expected")
    out = torch.empty(1, 1, H, dv, dtype=torch.bfloat16, device=query.device)
    with on_device(query.device):
        rc = lib().qfn_deltanet_step(query.data_ptr(), key.data_ptr(), value.data_ptr(), g.data_ptr(),
                                     beta.data_ptr(), initial_state.data_ptr(), out.data_ptr(), H, Hq, dk, dv,
                                     stream_of(out))
    check(rc, "qfn_deltanet_step")
    return out, initial_state


def chunk_gated_delta_rule(query, key, value, g, beta, initial_state=None, cu_seqlens=None, final_state=None,
                           out=None):
    """The gated delta rule over whole sequences -> (out, final_state).

    query, key [B, T, Hq, dk] bf16 (dk 64, 128 or 256) . value [B, T, H, dv] bf16
    (dv a multiple of 32, H a multiple of Hq) . g [B, T, H] fp32 (log of the
    decay; -inf clears the state) . beta [B, T, H] bf16 -> out [B, T, H, dv]
    bf16 and final_state [N, H, dk, dv] fp32.

    Without cu_seqlens the N = B rows of the batch are the sequences.  With it
    (int32 [N + 1] on the device, rising from >= 0 to <= T; B must be 1) sequence n
    is the tokens cu_seqlens[n] up to cu_seqlens[n + 1]; rows of out outside every
    sequence are left as they were.  Bounds that do not rise leave out unwritten
    and every final state NaN.  A sequence may have no token (its state passes
    through).

    initial_state [N, H, dk, dv] fp32 (None: zeros).  final_state and out may be
    given to be written; final_state may be initial_state itself.  Views of query,
    key, value, g and beta with any row and head strides are taken as they are;
    states start on 16 bytes, a given out on 4."""
    o, S = op("deltanet_chunk")(query, key, value, g, beta, cu_seqlens, initial_state, final_state, out)
    return o if out is None else out, S if final_state is None else final_state


def step_gated_delta_rule(query, key, value, g, beta, state, state_index=None, out_state=None, out=None):
    """One token of the gated delta rule for each of R requests -> (out, out_state).

    query, key [R, Hq, dk] bf16 . value [R, H, dv] bf16 . g [R, H] fp32 . beta
    [R, H] bf16 . state [slots, H, dk, dv] fp32 -> out [R, H, dv] bf16.

    Row r's state is state[state_index[r]] (int32 [R] on the device; None: slot
    r).  A negative index is a padding row: its out is zero and no state is
    touched.  An index past the pool, or one that an earlier row names too, gives NaN in
    that row's out and touches no state.  The new states are written to the same slots of out_state
    (None: state itself, in place); slots that no row names are left as they were.
    States start on 16 bytes."""
    if out_state is None:
        out_state = state
    o = op("deltanet_step")(query, key, value, g, beta, state, state_index, out_state, out)
    return o if out is None else out, out_state
