"""clip_gradients where its norm or its factor leaves fp32's range, and where its
partial sums are more than one kernel adds by itself, against float64
(tests/test_gpu_clip_gradients.py derives the bounds)."""
import math

import pytest
import torch

from neutrongt_amd import clip_gradients, gradient_norm
from tests.test_gpu_clip_gradients import BF16, F32, HALF, U, _check, _norm, _params, node  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("apart", [False, True])
def test_a_norm_that_fp32_cannot_hold_scales_nothing(dev, node, dtype, apart):
    """Two gradients of 3e38 have a norm of 4.2e38: returned as an infinity, so nothing is
    scaled; one of them alone is."""
    grads = [torch.full((2,), 3e38, dtype=dtype, device=dev), torch.ones(50, device=dev)]
    before = [t.clone() for t in grads]
    out = [torch.zeros_like(t) for t in grads] if apart else None
    assert clip_gradients(_params(grads), 1.0, out=out).item() == math.inf
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert not apart or all(torch.equal(a, b) for a, b in zip(out, before))
    assert gradient_norm(_params(grads)).item() == math.inf
    grads[0][1] = 0.0
    before, norm = [t.clone() for t in grads], _norm(grads)
    got = clip_gradients(_params(grads), 1.0, out=out)
    assert math.isfinite(got.item()) and abs(got.item() - norm) <= 1.01 * U * norm
    _check(out or grads, before, 1.0 / norm)


@pytest.mark.parametrize("dtype,out_dtype", [(F32, None), (BF16, None), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("size,limit", [(1e30, 1e-30), (3e38, 1e-2), (3e38, 3.0), (2e38, 1e-38),
                                        (1e20, 1e-20), (1e20, 1e-300)])
def test_a_factor_below_the_range_of_fp32(dev, node, size, limit, dtype, out_dtype):
    """Besides its roundings a result may be off by what its type's subnormal numbers, 2^-149
    and 2^-133 apart, lose: two halves of that, of the product and of its shift."""
    grads = [torch.tensor([size, -size / 3, size * 1e-7, 1.0, 0.0] * 3 + [0.5 * size], dtype=dtype,
                          device=dev) * 0.25, torch.ones(3, dtype=dtype, device=dev)]
    before, norm = [t.clone() for t in grads], _norm(grads)
    out = [torch.full_like(t, 7.0, dtype=out_dtype) for t in grads] if out_dtype else None
    got = clip_gradients(_params(grads), limit, out=out)
    assert abs(got.item() - norm) <= 1.01 * U * norm
    for t, g in zip(out or grads, before):
        want = g.double().cpu() * (limit / norm)
        half = HALF[t.dtype]
        bound = want.abs() * (2.1 * U + half * (1 + 2.1 * U)) + (2.0 ** -149 if t.dtype == F32 else 2.0 ** -133)
        assert ((t.double().cpu() - want).abs() <= bound).all()


def _apart(dev, count, size, dtype, seed):
    """Gradients in memory of their own each, as autograd makes them, all of other sizes."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(size + i % 3, device=dev, generator=g).to(dtype) for i in range(count)]


# one sum each of 2,500 tensors; 3,200 sums of two launches of 2,000 and 1,200 blocks
@pytest.mark.parametrize("dtype,out_dtype", [(F32, None), (BF16, None), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("count,size", [(2500, 1), (400, 60000)])
def test_more_sums_than_a_block_adds(dev, node, count, size, dtype, out_dtype):
    grads = _apart(dev, count, size, dtype, count)
    before, norm, ps = [t.clone() for t in grads], _norm(grads), _params(grads)
    assert abs(gradient_norm(ps).item() - norm) <= 1.01 * U * norm
    out = [torch.empty_like(t, dtype=out_dtype) for t in grads] if out_dtype else None
    for limit in (2 * norm, 0.25 * norm):
        got = clip_gradients(ps, limit, out=out)
        assert abs(got.item() - norm) <= 1.01 * U * norm
        _check(out or grads, before, min(1.0, limit / norm))
        if out or limit > norm:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))
    for bad in (math.nan, math.inf):
        for t, b in zip(grads, before):
            t.copy_(b)
        grads[count // 2][0] = bad
        assert not math.isfinite(clip_gradients(ps, 0.5, out=out).item())
        for t, b in zip(out or grads, before):
            if t is not (out or grads)[count // 2]:
                assert torch.equal(t, b.to(t.dtype))


def test_more_sums_than_a_block_adds_captured(dev, node):
    grads = _apart(dev, 2300, 5, F32, 1)
    ps = _params(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(ps, 1.0)
    for i in range(3):
        for t in grads:
            t.normal_().mul_(i + 1)
        before, want = [t.clone() for t in grads], _norm(grads)
        other = clip_gradients(_params([t.clone() for t in grads]), 1.0)  # eager work between
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, other) and abs(norm.item() - want) <= 1.01 * U * want
        _check(grads, before, 1 / want)


@pytest.mark.parametrize("count", [10, 2500])
def test_some_results_in_their_gradients_memory(dev, node, count):
    grads = _apart(dev, count, 9, F32, count)
    before, norm = [t.clone() for t in grads], _norm(grads)
    out = [t if i % 2 else torch.empty_like(t, dtype=BF16) for i, t in enumerate(grads)]
    for limit in (2 * norm, 0.5 * norm):
        got = clip_gradients(_params(grads), limit, out=out)
        assert abs(got.item() - norm) <= 1.01 * U * norm
        _check(out, before, min(1.0, limit / norm))
    assert all(torch.equal(a, b) for a, b in zip(grads[::2], before[::2]))
