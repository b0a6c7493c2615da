"""GELU and its derivative far below zero, where the result is as small as the normal
distribution's tail: each within its rounding to bf16 (a half step is at most 2^-8 of
it) and 2^-15 of it, not merely within a share of z.

The kernel's distribution is within 1e-5 of its value down to z = -13.  gelu' there is
Phi - |z| phi with |z| phi > 4 Phi from z = -2 on, so that the error of either is at most
1.7 times as large in it: 1.7e-5 < 2^-15."""
import math

import pytest
import torch

from neutrongt_amd import linear_epilogue

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("rows", [1, 200])  # 32 x 32 blocks, and the same z in many rows
def test_tail(dev, rows):
    z = (-torch.arange(2.0, 12.5, 0.03125)).to(BF16).unique()
    x = z.double()
    cdf = 0.5 * torch.erfc(-x / math.sqrt(2))
    phi = torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    n = z.numel()
    weight = torch.diag(z.float()).to(BF16).to(dev)  # z in column i from x = 1
    one = torch.ones(rows, n, dtype=BF16, device=dev).requires_grad_()
    bias = torch.zeros(n, dtype=BF16, device=dev).requires_grad_()
    y = linear_epilogue(one, weight, bias, "gelu")
    half = 2.0 ** -8 + 2.0 ** -15
    err = (y.detach().double().cpu() - x * cdf).abs() / (x * cdf).abs()
    assert err.max() <= half, f"gelu {err.max():.2e} at {z[err.max(0)[0].argmax()]}"
    # each gradient of the bias is one element of dz where the others' output gradient is 0
    gy = torch.zeros(rows, n, dtype=BF16, device=dev)
    gy[0] = 1.0
    db, = torch.autograd.grad(y, bias, gy)
    want = cdf + x * phi
    err = (db.double().cpu() - want).abs() / want.abs()
    assert err.max() <= half, f"gelu' {err.max():.2e} at {z[err.argmax()]}"


def test_tail_through_tiles(dev):
    """The same through whole 128 x 128 tiles."""
    z = (-torch.arange(2.0, 12.5, 0.03125)).to(BF16).unique()
    x = z.double()
    want = x * 0.5 * torch.erfc(-x / math.sqrt(2))
    rows = torch.cat([z] * 16)
    w = torch.zeros(1024, 64, dtype=BF16, device=dev)
    w[:, 0] = 1.0
    a = torch.zeros(rows.numel(), 64, dtype=BF16, device=dev)
    a[:, 0] = rows.to(dev)
    y = linear_epilogue(a, w, None, "gelu").double().cpu()
    ref = torch.cat([want] * 16)[:, None]
    assert ((y - ref).abs() <= (2.0 ** -8 + 2.0 ** -15) * ref.abs()).all()
