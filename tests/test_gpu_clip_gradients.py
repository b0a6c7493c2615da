"""clip_gradients and gradient_norm against float64.

The norm is summed in fp64 (n additions: n 2^-53 of it, below 2^-30 here) and rounded to
fp32 once: off by at most 1.01 u of itself, u = 2^-24.  The factor max_norm / norm is
rounded to fp32 (u), the product too (u), then the result to its type: 2.1 u and the
type's half step."""
import math

import pytest
import torch

from neutrongt_amd import _lib, clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(params=["cpp", "python"])
def node(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    else:
        assert _lib.autograd_ext() is not None


def _params(grads):
    ps = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        ps.append(p)
    return ps


def _norm(grads):
    return math.sqrt(sum(float((g.double().cpu() ** 2).sum()) for g in grads))


def _check(got, before, by):
    for t, g in zip(got, before):
        want = g.double().cpu() * by
        bound = want.abs() * (2.1 * U + HALF[t.dtype] * (1 + 2.1 * U)) + 2.0 ** -149
        assert ((t.double().cpu() - want).abs() <= bound).all()


SHAPES = [[(3,)], [(1,)], [(64, 64), (64,), (7, 3), (1,)], [(5, 7, 3)] * 200, [(1 << 14,)],
          [((1 << 14) + 1,), ((1 << 15) - 3,)], [(1000, 1001), (4,), (0,), (3, 0)],
          [(3000001,), (17,)]]


@pytest.mark.parametrize("dtype,out_dtype", [(F32, None), (BF16, None), (BF16, F32), (F32, BF16),
                                             (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("shapes", range(len(SHAPES)))
def test_norm_and_clip(dev, node, shapes, dtype, out_dtype):
    print(f"case {SHAPES[shapes][:4]} {dtype} {out_dtype}", flush=True)
    g = torch.Generator().manual_seed(shapes)
    grads = [torch.randn(s, generator=g).to(dtype).to(dev) for s in SHAPES[shapes]]
    before = [t.clone() for t in grads]
    norm = _norm(grads)
    ps = _params(grads)
    got = gradient_norm(ps)
    assert got.shape == () and got.dtype == F32 and abs(got.item() - norm) <= 1.01 * U * norm
    out = [torch.empty_like(t, dtype=out_dtype) for t in grads] if out_dtype else None
    for limit in (2 * norm, 0.25 * norm, 0.0):
        for t, b in zip(grads, before):
            t.copy_(b)
        got = clip_gradients(ps, limit, out=out)
        assert abs(got.item() - norm) <= 1.01 * U * norm
        _check(out or grads, before, min(1.0, limit / norm))
        if out:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))
        elif limit > norm:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_mixed_types_orders_and_alignment(dev, node):
    g = torch.Generator().manual_seed(1)
    flat = torch.randn(5000, generator=g).to(dev)
    grads = [flat[1:1001].view(10, 100), flat[1001:1004], flat[1008:1008 + 48].view(6, 8).t(),
             torch.randn(30, 20, 4, generator=g).to(BF16).to(dev).permute(2, 0, 1),
             torch.randn(4, 3, 8, 8, generator=g).to(dev).to(memory_format=torch.channels_last),
             torch.randn(999, generator=g).to(BF16).to(dev)[5:], torch.tensor(3.0, device=dev),
             torch.randn(1, 7, generator=g).to(dev).as_strided((1, 7), (99, 1))]
    before, norm = [t.clone() for t in grads], _norm(grads)
    rest = flat.clone()
    got = clip_gradients(_params(grads), 0.1)
    assert abs(got.item() - norm) <= 1.01 * U * norm
    _check(grads, before, 0.1 / norm)
    seen = torch.zeros(5000, dtype=torch.bool, device=dev)
    seen[1:1004] = seen[1008:1056] = True
    assert torch.equal(flat[~seen], rest[~seen])  # what lies between is left alone


def test_a_result_in_its_gradients_own_memory(dev, node):
    grads = [torch.full((100,), 2.0, device=dev), torch.full((33,), -1.0, device=dev)]
    before, norm = [t.clone() for t in grads], _norm(grads)
    ps = _params(grads)
    clip_gradients(ps, 1.0, out=grads)
    _check(grads, before, 1 / norm)


def test_a_parameter_twice_and_without_gradient(dev, node):
    ps = _params([torch.full((10,), 3.0, device=dev), torch.full((4,), 4.0, device=dev)])
    none = torch.nn.Parameter(torch.zeros(5, device=dev))
    got = clip_gradients([ps[0], none, ps[1], ps[0]], 1.0)
    norm = math.sqrt(90 + 64)
    assert abs(got.item() - norm) <= 1.01 * U * norm and none.grad is None
    _check([p.grad for p in ps], [torch.full((10,), 3.0), torch.full((4,), 4.0)], 1 / norm)
    assert clip_gradients(ps[0], 1e9).item() == pytest.approx(3 * math.sqrt(10) / norm, rel=1e-6)
    assert clip_gradients([none], 1.0).item() == 0.0
    assert gradient_norm([]).item() == 0.0
    assert clip_gradients((p for p in ps), 1e9).item() > 0  # a generator


def test_a_norm_that_is_not_finite_scales_nothing(dev, node):
    for bad in (math.inf, -math.inf, math.nan):
        grads = [torch.randn(1000, device=dev), torch.randn(50, device=dev).to(BF16)]
        grads[0][77] = bad
        before = [t.clone() for t in grads]
        got = clip_gradients(_params(grads), 0.5)
        assert not math.isfinite(got.item())
        assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(grads, before))


def test_squares_that_fp32_cannot_hold(dev, node):
    for size in (1e30, 1e-30):
        grads = [torch.full((300,), size, device=dev), torch.full((100,), -size, device=dev)]
        got = clip_gradients(_params(grads), size)
        assert abs(got.item() - 20 * size) <= 1e-6 * 20 * size
        assert torch.allclose(grads[0], torch.full_like(grads[0], size / 20), rtol=1e-6, atol=0)


def test_more_tensors_than_a_launch_takes(dev, node):
    grads = [torch.full((i % 7 + 1,), 1.0 + i % 3, device=dev) for i in range(1000)]
    before, norm = [t.clone() for t in grads], _norm(grads)
    got = clip_gradients(_params(grads), 1.0)
    assert abs(got.item() - norm) <= 1.01 * U * norm
    _check(grads, before, 1 / norm)


def test_offsets_behind_2_to_the_31(dev):
    n = (1 << 31) + 12345
    t = torch.zeros(n, dtype=BF16, device=dev)
    t[-1], t[1 << 31], t[0] = 3.0, 4.0, 12.0
    p, = _params([t])
    assert gradient_norm(p).item() == 13.0
    assert clip_gradients(p, 6.5).item() == 13.0
    assert [t[i].item() for i in (-1, 1 << 31, 0)] == [1.5, 2.0, 6.0] and t.sum().item() == 9.5


def test_the_version_counts_and_the_bits_are_the_same_every_time(dev, node):
    w = torch.randn(300, 300, device=dev, requires_grad=True)
    x = torch.randn(300, 300, device=dev, requires_grad=True)
    w.grad = torch.randn(300, 300, device=dev)
    y = (x * w.grad).sum()  # the graph keeps the gradient
    clip_gradients(w, 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    g = [torch.randn(100003, device=dev), torch.randn(7, device=dev)]
    a, b = ([t.clone() for t in g] for _ in range(2))
    na, nb = clip_gradients(_params(a), 1.0), clip_gradients(_params(b), 1.0)
    assert torch.equal(na, nb) and all(torch.equal(s, t) for s, t in zip(a, b))


def test_captured_and_on_another_stream(dev, node):
    grads = [torch.randn(50000, device=dev), torch.randn(333, 9, device=dev).to(BF16)]
    ps = _params(grads)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        first = clip_gradients(ps, 1e9)
    side.synchronize()
    assert abs(first.item() - _norm(grads)) <= 1.01 * U * first.item()
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


def test_refusals(dev, node):
    one = lambda *s, **k: torch.ones(*s, device=dev, **k)
    flat = one(100)
    for grads, kw, err in (
            ([one(3).cpu()], {}, ValueError), ([one(3), one(3).cpu()], {}, ValueError),
            ([one(3).half()], {}, TypeError), ([one(3, dtype=torch.float64)], {}, TypeError),
            ([one(3, 4)[:, :2]], {}, ValueError), ([one(1, 4).expand(3, 4)], {}, ValueError),
            ([flat[:10], flat[5:20]], {}, ValueError), ([flat[:50], flat[3:5], flat[60:]], {}, ValueError),
            ([flat[:10]], dict(out=[flat[4:14]]), ValueError),
            ([flat[:10], flat[10:20]], dict(out=[flat[10:20], flat[:10]]), ValueError),
            ([one(4)], dict(out=[]), ValueError), ([one(4)], dict(out=[one(5)]), ValueError),
            ([one(4)], dict(out=[one(4).half()]), TypeError),
            ([one(3, 4)], dict(out=[one(4, 3).t()]), ValueError),
            ([one(3, 4).to_sparse()], {}, ValueError)):
        ps = []
        for g in grads:
            p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device))
            p.grad = g
            ps.append(p)
        with pytest.raises(err):
            clip_gradients(ps, 0.1, **kw)
    ps = _params([one(4)])
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            clip_gradients(ps, bad)
    assert torch.equal(ps[0].grad, one(4))
