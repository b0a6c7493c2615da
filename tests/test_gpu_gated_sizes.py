"""gated_linear at sizes whose helping launches (rows filled up to whole pieces, the joins)
have more to do than a launch takes blocks.  Rows of zeros give zeros and add nothing to the
weights' gradients, so float64 is needed for the rows alone that hold something
(tests/test_gpu_gated_linear.py derives the bounds)."""
import pytest
import torch

from neutrongt_amd import gated_linear
from tests.test_gpu_gated_linear import BF16, _check, _inputs, _ref

pytestmark = pytest.mark.gpu


def _rows(dev, M, N, K, at, seed):
    """x [M, K] of zeros but for the rows `at`, and what stands there."""
    some, wg, wu, _, _, gy = _inputs(len(at), N, K, False, seed)
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    x[torch.tensor(at, device=dev)] = some.to(dev)
    return x, wg.to(dev), wu.to(dev), gy, _ref(some, wg, wu, None, None, gy, "silu")


def _others_are_zero(t, at):
    t = t.detach().clone()
    t[torch.tensor(at, device=t.device)] = 0
    return not any(bool(c.any()) for c in t.split(1 << 20))


def test_filled_up_rows_that_share_blocks(dev):
    M, K, at = (1 << 20) + 77, 1025, [0, 1, 76, 77, (1 << 20) - 1, 1 << 20, (1 << 20) + 76]
    for N in (8, 232):
        print(f"case M={M} N={N} K={K}", flush=True)
        x, wg, wu, some_gy, ref = _rows(dev, M, N, K, at, N)
        gy = torch.ones(M, N, dtype=BF16, device=dev)
        gy[torch.tensor(at, device=dev)] = some_gy.to(dev)
        leaves = [t.requires_grad_() for t in (x, wg, wu)]
        y = gated_linear(*leaves)
        dx, dg, du = torch.autograd.grad(y, leaves, gy)
        _check([y[at].detach(), dx[at], dg, du], ref, "gated")
        assert _others_are_zero(y, at) and _others_are_zero(dx, at)


def test_as_many_filled_up_rows_as_a_launch_has_blocks_at_most(dev):
    """2^24 rows of 1,025, of which a block takes one at a time, are 2^32 threads."""
    M, N, K = 1 << 24, 256, 1025
    at = [0, 12345678, M - 2, M - 1]
    x, wg, wu, _, ref = _rows(dev, M, N, K, at, 1)
    with torch.no_grad():
        y = gated_linear(x, wg, wu)
    _check([y[at]], ref[:1], "gated")
    assert _others_are_zero(y, at)
    del x, y
    torch.cuda.empty_cache()


def test_weights_of_more_sums_than_a_launch_has_threads(dev):
    """The join of two weights of 2^33 elements, 4 a thread, would be 2^32 threads.  No rows:
    all of the gradient is written as zeros."""
    N, K = 1 << 16, 1 << 17
    w = torch.empty(N, K, dtype=BF16, device=dev).requires_grad_()
    x = torch.empty(0, K, dtype=BF16, device=dev)
    filler = torch.full((N, K), 3.0, dtype=BF16, device=dev)
    del filler  # the gradient's memory, most likely, holds something
    y = gated_linear(x, w, w.detach())
    dw, = torch.autograd.grad(y, w, torch.empty_like(y))
    assert dw.shape == (N, K) and not any(bool(c.any()) for c in dw.split(1 << 12))
    del dw, w, x, y
    torch.cuda.empty_cache()


def test_weights_whose_joined_sums_share_blocks(dev):
    """2 x 66,000 x 8,193 sums of odd rows, 1,024 a block, are more than 2^20 blocks."""
    M, N, K = 3, 66000, 8193
    x, wg, wu, _, _, gy = _inputs(M, 1, K, False, 5)
    gy = torch.randn(M, N, generator=torch.Generator().manual_seed(6)).to(BF16)
    g = torch.Generator(device=dev).manual_seed(7)
    wg, wu = (torch.randn(N, K, device=dev, dtype=BF16, generator=g).mul_(K ** -0.5).requires_grad_()
              for _ in range(2))
    dg, du = torch.autograd.grad(gated_linear(x.to(dev), wg, wu), (wg, wu), gy.to(dev))
    with torch.device(dev):  # the reference on the GPU, for its size
        ref = _ref(x.to(dev), wg.detach(), wu.detach(), None, None, gy.to(dev), "silu")
    for got, (want, bound) in zip((dg, du), ref[2:4]):
        assert ((got.double() - want).abs() <= bound).all()
    del ref, want, bound
    torch.cuda.empty_cache()
