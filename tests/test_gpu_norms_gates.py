"""The gates of norms.gated_rms_norm and norms.norm_residual over the whole range of the sigmoid, against 64 bits.

Tolerances: one rounding of the output (2^-8 of the value for bf16, 2^-24 for fp32), and the gate's own: the product
x log2(e) is rounded to 2^-24 of a number up to 151 (beyond it the exponential is below 2^-149), which moves the
exponential by 151 ln 2 2^-24 < 2^-17, the dozen roundings of the rest by less than 2^-20: 2^-16 in all.  Below 2^-126 an
exponential has steps of 2^-149, so that a product with a factor f is off by f 2^-149: f = 2^20 in the residual's
cases, and 2^20 |z| <= 2^27 in the gated norm's, 2^-129 and 2^-122.
"""
import pytest
import torch

import norms

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LOWEST = torch.finfo(torch.bfloat16).min


def near(got, want, floor):
    err = (got.double() - want).abs()
    lim = (HALF_STEP[got.dtype] + 2.0 ** -16) * want.abs() + floor
    assert (err <= lim).all(), f"{(err / lim).max():.2f} x tolerance"


def gates(n):
    """bf16 values from -128 to 128, dense around zero and where the sigmoid's reciprocal leaves fp32's normal numbers."""
    z = torch.cat([torch.linspace(-128, 128, 1025), torch.linspace(-4, 4, 513), torch.linspace(-104, -80, 97)])
    return z.to(torch.bfloat16).to(DEV)[:n]


@pytest.mark.parametrize("D", [64, 96, 100, 320])
def test_gated_norm_gate(D):
    z = gates(1635 // D * D).view(-1, 1, D)
    x = torch.ones_like(z)
    w = torch.full((D,), 2.0 ** 20, device=DEV)
    y = norms.gated_rms_norm(x, z, w, eps=0.0)
    zd = z.double()
    near(y, 2.0 ** 20 * zd * torch.sigmoid(zd), 2.0 ** -122)
    odd = torch.empty(z.shape[0], 1, D + 1, dtype=z.dtype, device=DEV)[:, :, 1:]   # off 16 bytes
    odd.copy_(z)
    near(norms.gated_rms_norm(x, odd, w, eps=0.0), 2.0 ** 20 * zd * torch.sigmoid(zd), 2.0 ** -122)


@pytest.mark.parametrize("D", [64, 65, 66, 4104])
@pytest.mark.parametrize("gd", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_row", [False, True])
def test_residual_gate(per_row, gd, D):
    z = gates(1635).to(gd)
    gate = z[:, None] if per_row else z[None, :].expand(3, -1).repeat(1, -(-3 * D // z.numel()))[:, :D].contiguous()
    block = torch.full((gate.shape[0], D), 2.0 ** 20, device=DEV)
    zero = torch.zeros(gate.shape[0], D, device=DEV)
    r, _ = norms.norm_residual(block, zero, gate=gate)
    near(r, (2.0 ** 20 * torch.sigmoid(gate.double())).expand(-1, D), 2.0 ** -129)
    r, _ = norms.norm_residual(block, zero, gate=gate, sigmoid=False)
    near(r, (2.0 ** 20 * gate.double()).expand(-1, D), 2.0 ** -129)


def test_gate_ends():
    """Zero, the lowest and highest values, infinities and NaN."""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([0.0, -0.0, LOWEST, -LOWEST, -inf, inf, nan, 1.0], dtype=torch.bfloat16, device=DEV)[:, None]
    block, zero = torch.ones(8, 64, device=DEV), torch.zeros(8, 64, device=DEV)
    r, _ = norms.norm_residual(block, zero, gate=z)
    want = torch.tensor([0.5, 0.5, 0, 1, 0, 1, nan, torch.sigmoid(torch.tensor(1.0)).item()], device=DEV)
    assert torch.allclose(r[:, 0], want, rtol=2.0 ** -20, atol=0, equal_nan=True)
