"""The operators of a linear-attention layer between its quantized products, as
cases to measure: the gated delta rule over prompts (deltanet.chunk_gated_delta_rule)
and over a batch of single tokens (deltanet.step_gated_delta_rule), the gated
norm of its output (norms.gated_rms_norm), and the norms around a block with
its gate and residual scale (norms.norm_residual).

`own` false computes them with elementary torch operations in 32 bits (the
chunk's cumulative decays in 64), true through the framework's entry points.
"""
import os
import sys

import torch

own = False

EPS = 1e-6
CHUNK = 64   # tokens of a chunk in the plain form
DEV = "cuda"


# ------------------------------------------------------------------ cases
# 32 heads of 128 x 128 are the layer that the FP8 projections of bench.py
# imply; with 16 key heads each serves two value heads.
def listed():
    big = {"heads": 32, "key_heads": 32, "dk": 128, "dv": 128}
    shared = {**big, "key_heads": 16}
    return [
        # a short question: one request, two full chunks and a ragged one
        {"name": "prompt-130", "op": "chunk", "lens": "130", **big, "carried": False},
        # the prompt piece of the headline benchmark
        {"name": "prompt-2048", "op": "chunk", "lens": "2048", **big, "carried": False},
        # a long document, continued from an earlier piece
        {"name": "prompt-16384", "op": "chunk", "lens": "16384", **big, "carried": True},
        # requests of a server taken together: ragged, one of them empty, one a single token
        {"name": "ragged-9", "op": "chunk", "lens": "611,1,64,0,1537,129,900,63,2050", **shared, "carried": True},
        # a shard of the heads on one of several GPUs, narrow keys
        {"name": "narrow-heads", "op": "chunk", "lens": "1000,3001", "heads": 8, "key_heads": 4, "dk": 64, "dv": 96,
         "carried": True},
        # one request, one token: latency
        {"name": "token-1", "op": "step", "rows": 1, "padding": 0, **big},
        # the batched-decode benchmark's 64 requests
        {"name": "tokens-64", "op": "step", "rows": 64, "padding": 0, **big},
        # a captured batch of 256 rows of which 19 are padding
        {"name": "tokens-256-padded", "op": "step", "rows": 256, "padding": 19, **shared},
        # the layer's output norm for a batch of 64 requests, and for a long prompt
        {"name": "gated-norm-64", "op": "gated_norm", "tokens": 64, "heads": 32, "dim": 128},
        {"name": "gated-norm-16384", "op": "gated_norm", "tokens": 16384, "heads": 32, "dim": 128},
        # around an MoE block (fp32 output, a gate for each token): one token, then a long prompt
        {"name": "residual-1", "op": "residual", "tokens": 1, "dim": 2560, "block_f32": True, "gate": "token"},
        {"name": "residual-16384", "op": "residual", "tokens": 16384, "dim": 2560, "block_f32": False,
         "gate": "channel"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "step", "gated_norm", "residual"])
    if op in ("chunk", "step"):
        heads = rng.choice([4, 8, 12, 16, 24, 32])
        d = {"op": op, "heads": heads, "key_heads": heads // rng.choice([1, 2, 4]), "dk": rng.choice([64, 128]),
             "dv": rng.choice([32, 64, 96, 128])}
        if op == "chunk":
            n = _log(rng, 1, 16)
            lens = [0 if n > 1 and rng.random() < 0.1 else _log(rng, 1, 16384 // n) for _ in range(n)]
            lens[rng.randrange(n)] = _log(rng, 16, 16384 // n)
            return {**d, "lens": ",".join(map(str, lens)), "carried": rng.random() < 0.5}
        rows = _log(rng, 1, 256)
        return {**d, "rows": rows, "padding": rng.randrange(1 + rows // 8)}
    if op == "gated_norm":
        return {"op": op, "tokens": _log(rng, 1, 16384), "heads": rng.choice([4, 8, 16, 32]),
                "dim": rng.choice([64, 96, 128])}
    return {"op": op, "tokens": _log(rng, 1, 16384), "dim": _log(rng, 300, 2560),
            "block_f32": rng.random() < 0.5, "gate": rng.choice(["none", "token", "channel"])}


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    op = case["op"]
    if op in ("chunk", "step"):
        H, Hk, dk, dv = case["heads"], case["key_heads"], case["dk"], case["dv"]
        T = sum(_lens(case)) if op == "chunk" else case["rows"]
        # one row per token holds q, k and v side by side, as the projection and its activation leave them
        qkv = torch.nn.functional.silu(normal(T, 2 * Hk * dk + H * dv)).to(torch.bfloat16)
        q, k, v = (t.view(T, -1, d) for t, d in zip(qkv.split([Hk * dk, Hk * dk, H * dv], 1), (dk, dk, dv)))
        a_log = torch.empty(H, device=DEV).uniform_(-2, 1, generator=gen)
        g = -a_log.exp() * torch.nn.functional.softplus(normal(T, H))
        beta = torch.sigmoid(normal(T, H)).to(torch.bfloat16)
        s = {"q": q, "k": k, "v": v, "g": g, "beta": beta}
        if op == "chunk":
            lens = _lens(case)
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + n)
            s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
            s["state"] = normal(len(lens), H, dk, dv) * 0.05 if case["carried"] else None
        else:
            slots = T
            live = T - case["padding"]
            index = torch.randperm(slots, device=DEV, generator=gen).to(torch.int32)
            index[live:] = -1
            s["index"] = index
            s["state"] = normal(slots, H, dk, dv) * 0.05
        return s
    if op == "gated_norm":
        T, H, D = case["tokens"], case["heads"], case["dim"]
        return {"x": normal(T, H, D).to(torch.bfloat16), "z": normal(T, H * D).to(torch.bfloat16).view(T, H, D),
                "w": 1 + 0.1 * normal(D)}
    T, D = case["tokens"], case["dim"]
    block = normal(T, D)
    gate = {"none": None, "token": (T, 1), "channel": (T, D)}[case["gate"]]
    return {"block": block if case["block_f32"] else block.to(torch.bfloat16),
            "residual": (3 * normal(T, D)).to(torch.bfloat16),
            "gate": None if gate is None else normal(*gate).to(torch.bfloat16),
            "post": (1 + 0.1 * normal(D)).to(torch.bfloat16), "next": (1 + 0.1 * normal(D)).to(torch.bfloat16),
            "scale": 0.7}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"] = case["op"]
    if case["op"] == "chunk":
        s["seqs"], s["longest"] = len(_lens(case)), max(_lens(case))   # known to a scheduler on the host
    elif case["op"] == "step":
        s["live"] = case["rows"] - case["padding"]
        s["out_state"] = torch.zeros_like(s["state"])
    return s


# ------------------------------------------------------------------ plain forms
def _l2(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular A [..., C, C], row by row."""
    C = A.shape[-1]
    X = torch.eye(C, device=A.device, dtype=A.dtype).expand(A.shape).contiguous()
    for i in range(1, C):
        X[..., i, :i] = -(A[..., i, None, :i] @ X[..., :i, :i])[..., 0, :]
    return X


def _chunk_plain(s):
    N, H = s["seqs"], s["v"].shape[1]
    Hk, dk, dv = s["q"].shape[1], s["q"].shape[2], s["v"].shape[2]
    C = CHUNK
    M = -(-s["longest"] // C)
    cu = s["cu"].long()
    pos = torch.arange(M * C, device=DEV)
    live = pos[None] < (cu[1:] - cu[:-1])[:, None]
    at = torch.where(live, cu[:-1, None] + pos[None], 0)

    def rows(x, heads):   # [T, heads, ...] -> fp32 [N, H, M, C, ...], zero behind a sequence's end
        x = x.float()[at] * live.view(N, -1, *[1] * (x.dim() - 1))
        x = x.view(N, M, C, *x.shape[2:])
        return x.movedim(3, 1).repeat_interleave(H // heads, 1)

    q, k, v = rows(s["q"], Hk), rows(s["k"], Hk), rows(s["v"], H)
    q, k = _l2(q) / dk ** 0.5, _l2(k)
    G = rows(s["g"], H).double().cumsum(-1)
    beta = rows(s["beta"], H)
    decay = (G[..., :, None] - G[..., None, :]).tril().exp().float().tril()
    X = _inverse((beta[..., None] * decay * (k @ k.transpose(-1, -2))).tril(-1))
    inner = decay * (q @ k.transpose(-1, -2))
    begin = G.exp().float()[..., None]
    end = (G[..., -1:] - G).exp().float()[..., None]
    last = G[..., -1].exp().float()[..., None, None]
    S = torch.zeros(N, H, dk, dv, device=DEV) if s["state"] is None else s["state"]
    o = torch.empty_like(v)
    for c in range(M):
        d = X[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - begin[:, :, c] * (k[:, :, c] @ S)))
        o[:, :, c] = begin[:, :, c] * (q[:, :, c] @ S) + inner[:, :, c] @ d
        S = last[:, :, c] * S + (end[:, :, c] * k[:, :, c]).transpose(-1, -2) @ d
    out = torch.empty(s["v"].shape[0], H, dv, device=DEV)
    flat = o.movedim(1, 3).reshape(N * M * C, H, dv)
    # every token's row among the padded ones
    token = torch.arange(out.shape[0], device=DEV)
    seq = (token[:, None] >= cu[None, 1:]).sum(1)
    out = flat[seq * (M * C) + token - cu[seq]]
    return {"out": out.to(torch.bfloat16)[None], "state": S}


def _step_plain(s):
    n, H, Hk = s["live"], s["v"].shape[1], s["q"].shape[1]
    dk = s["q"].shape[2]
    at = s["index"][:n].long()
    q = (_l2(s["q"][:n].float()) / dk ** 0.5).repeat_interleave(H // Hk, 1)
    k = _l2(s["k"][:n].float()).repeat_interleave(H // Hk, 1)
    S = s["state"][at] * s["g"][:n].exp()[..., None, None]
    d = (s["v"][:n].float() - (S * k[..., None]).sum(2)) * s["beta"][:n].float()[..., None]
    S = S + k[..., None] * d[:, :, None]
    s["out_state"][at] = S
    out = torch.zeros(s["v"].shape, device=DEV)
    out[:n] = (S * q[..., None]).sum(2)
    return {"out": out.to(torch.bfloat16), "state": s["out_state"]}


def _gated_norm_plain(s):
    x, z = s["x"].float(), s["z"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].float()
    return (y * z / (1 + torch.exp(-z))).to(torch.bfloat16)


def _residual_plain(s):
    b = s["block"].float()
    p = b * torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        p = p / (1 + torch.exp(-s["gate"].float()))
    r = s["residual"].float() + s["scale"] * p
    n = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * s["next"].float()
    return r.to(torch.bfloat16), n.to(torch.bfloat16)


PLAIN = {"chunk": _chunk_plain, "step": _step_plain, "gated_norm": _gated_norm_plain, "residual": _residual_plain}


# ------------------------------------------------------------------ the framework's calls
def _chunk_own(s):
    import deltanet
    o, S = deltanet.chunk_gated_delta_rule(s["q"][None], s["k"][None], s["v"][None], s["g"][None], s["beta"][None],
                                           initial_state=s["state"], cu_seqlens=s["cu"])
    return {"out": o, "state": S}


def _step_own(s):
    import deltanet
    o, S = deltanet.step_gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                                          state_index=s["index"], out_state=s["out_state"])
    return {"out": o, "state": S}


def _gated_norm_own(s):
    import norms
    return norms.gated_rms_norm(s["x"], s["z"], s["w"], eps=EPS)


def _residual_own(s):
    import norms
    return norms.norm_residual(s["block"], s["residual"], post_weight=s["post"], gate=s["gate"], scale=s["scale"],
                               next_weight=s["next"], eps=EPS)


OWN = {"chunk": _chunk_own, "step": _step_own, "gated_norm": _gated_norm_own, "residual": _residual_own}
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-flash-next-8gb_b200")


def run(state):
    if own:
        if PACKAGE not in sys.path:   # the framework's modules are top-level modules of this directory
            sys.path.insert(0, PACKAGE)
        return OWN[state["op"]](state)
    return PLAIN[state["op"]](state)


# ------------------------------------------------------------------ work and exact values
def work(case):
    op = case["op"]
    if op in ("chunk", "step"):
        H, Hk, dk, dv = case["heads"], case["key_heads"], case["dk"], case["dv"]
        row = 2 * (2 * Hk * dk + H * dv) + 6 * H + 2 * H * dv   # q, k, v, g, beta in; out
        S = 4 * H * dk * dv
        if op == "chunk":
            lens = _lens(case)
            T = sum(lens)
            return {"bytes": T * row + len(lens) * S * (2 if case["carried"] else 1) + 4 * (len(lens) + 1),
                    "flops": 6 * T * H * dk * dv}
        n = case["rows"] - case["padding"]
        return {"bytes": n * (row + 2 * S) + 4 * case["rows"], "flops": 7 * n * H * dk * dv}
    if op == "gated_norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 6 * n + 4 * case["dim"], "flops": 12 * n}
    T, D = case["tokens"], case["dim"]
    gate = {"none": 0, "token": 2 * T, "channel": 2 * T * D}[case["gate"]]
    return {"bytes": T * D * ((4 if case["block_f32"] else 2) + 2 + 2 + 2) + gate + 4 * D, "flops": 14 * T * D}


def _token64(S, q, k, v, g, beta):
    """One token of the gated delta rule in 64 bits: S [..., dk, dv] -> (out, new S)."""
    q = q / ((q * q).sum(-1, keepdim=True) + EPS).sqrt() / q.shape[-1] ** 0.5
    k = k / ((k * k).sum(-1, keepdim=True) + EPS).sqrt()
    S = S * g.exp()[..., None, None]
    d = beta[..., None] * (v - torch.einsum("...kv,...k->...v", S, k))
    S = S + torch.einsum("...k,...v->...kv", k, d)
    return torch.einsum("...kv,...k->...v", S, q), S


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("chunk", "step"):
        r = case["heads"] // case["key_heads"]
        q, k = s["q"].double().repeat_interleave(r, 1), s["k"].double().repeat_interleave(r, 1)
        v, g, beta = s["v"].double(), s["g"].double(), s["beta"].double()
        if op == "step":
            n = case["rows"] - case["padding"]
            at = s["index"][:n].long()
            o, S = _token64(s["state"][at].double(), q[:n], k[:n], v[:n], g[:n], beta[:n])
            out, state = torch.zeros_like(v), torch.zeros(s["state"].shape, dtype=torch.float64, device=DEV)
            out[:n], state[at] = o, S
            return {"out": out, "state": state}
        lens, cu = _lens(case), s["cu"].tolist()
        S = torch.zeros(len(lens), case["heads"], case["dk"], case["dv"], dtype=torch.float64, device=DEV)
        if s["state"] is not None:
            S += s["state"]
        out = torch.zeros_like(v)
        # the longest first: the sequences that have a t-th token are then a leading part
        order = sorted(range(len(lens)), key=lambda i: -lens[i])
        start = torch.tensor([cu[i] for i in order], device=DEV)
        P = S[order]
        for t in range(max(lens)):
            m = sum(lens[i] > t for i in order)
            at = start[:m] + t
            out[at], P[:m] = _token64(P[:m], q[at], k[at], v[at], g[at], beta[at])
        S[order] = P
        return {"out": out[None], "state": S}
    if op == "gated_norm":
        x, z = s["x"].double(), s["z"].double()
        y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        return y * s["w"].double() * z * torch.sigmoid(z)
    b = s["block"].double()
    p = b / (b.square().mean(-1, keepdim=True) + EPS).sqrt() * s["post"].double()
    if s["gate"] is not None:
        p = p * torch.sigmoid(s["gate"].double())
    r = s["residual"].double() + s["scale"] * p
    return r, r / (r.square().mean(-1, keepdim=True) + EPS).sqrt() * s["next"].double()
