"""Norms of a layer around its blocks, fused with the gate, the residual scale and
the residual add that follow them (libqfn's qfn_gated_norm and
qfn_norm_residual).

RMSNorm here is x * rsqrt(mean(x^2) + eps) * weight, computed in fp32; every
output is rounded once.  Both are forward only and refuse a tensor that requires
a gradient while gradients are recorded.
"""
from _lib import op


def gated_rms_norm(x, z, weight, eps=1e-6):
    """rmsnorm(x) * weight * silu(z) over the last dimension -> bf16, x's shape:
    the norm of the linear attention's heads with the output gate.

    x, z [..., H, D] or [T, D] bf16 (views with any strides of rows and heads) .
    weight [D] bf16 or fp32."""
    if x.dim() < 2 or z.shape != x.shape:
        raise ValueError(f"x and z must have the same shape of two or more dimensions, got {tuple(x.shape)}, "
                         f"{tuple(z.shape)}")
    if x.dim() == 2:
        return op("gated_norm")(x[:, None], z[:, None], weight, eps)[:, 0]
    if x.dim() == 3:
        return op("gated_norm")(x, z, weight, eps)
    return op("gated_norm")(x.flatten(0, -3), z.flatten(0, -3), weight, eps).view(x.shape)


def norm_residual(block, residual, post_weight=None, gate=None, scale=1.0, next_weight=None, eps=1e-6,
                  sigmoid=True, out=None):
    """What stands between two blocks, in one pass -> (new residual, next block's input):

        p = rmsnorm(block) * post_weight                  (block itself without post_weight)
        r = residual + scale * sigmoid(gate) * p          (gate itself with sigmoid=False; 1 without gate)
        n = rmsnorm(r) * next_weight                      (None without next_weight)

    block [T, D] bf16 or fp32 . residual [T, D] bf16 or fp32 . gate [T], [T, 1] or
    [T, D] bf16 or fp32 . weights [D] bf16 or fp32, D <= 32768 -> r in residual's
    type, n bf16.  n is formed from r before its rounding.  out: where r goes, residual itself included."""
    if gate is not None and gate.dim() == 1:
        gate = gate[:, None]
    r, n = op("norm_residual")(block, residual, post_weight, gate, sigmoid, scale, next_weight, eps, out)
    return r if out is None else out, None if next_weight is None else n
