"""linear_epilogue against float64: y = act(x W^T + b) + r and its gradients, each
element within the bound of the roundings made.

The products of bf16 values are exact in fp32 (u = 2^-24 its half step, h = 2^-8
bf16's), a sum of n of them is off by at most n u of their absolute values.
  z:   e_z = (K + 2) u (sum|x||w| + |b|)
  y:   1.13 e_z (gelu's slope is at most 1.13) + 8 u (|z| + |act| + |r|), then h |y|
  dz:  |g| times act' of z rounded to bf16: gelu'' is at most 0.8, relu' may
       differ where |z| <= e_z; then h |dz|
  dx, dw, db: sums of dz's error and n u of the terms, then h (bf16) or nothing"""
import math

import pytest
import torch

from neutrongt_amd import _lib, linear_epilogue
from neutrongt_amd.linear import ACTIVATIONS

pytestmark = pytest.mark.gpu
U, HB = 2.0 ** -24, 2.0 ** -8
BF16, F32 = torch.bfloat16, torch.float32


def _ref(x, w, b, r, gy, act, w_type=BF16):
    x, w, gy = x.double(), w.double(), gy.double()
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    bb = b.double() if b is not None else torch.zeros(N, dtype=torch.float64)
    rr = r.double() if r is not None else torch.zeros(M, N, dtype=torch.float64)
    z = x @ w.t() + bb
    ez = (K + 2) * U * (x.abs() @ w.abs().t() + bb.abs())
    cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    a = z * cdf if act == "gelu" else z.clamp(min=0) if act == "relu" else z
    y = a + rr
    ey = 1.13 * ez + 8 * U * (z.abs() + a.abs() + rr.abs())
    da = (cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi) if act == "gelu"
          else (z > 0).double() if act == "relu" else torch.ones_like(z))
    dz = gy * da
    e = (gy.abs() * (0.8 * (ez + HB * (z.abs() + ez)) + 16 * U) if act == "gelu"
         else gy.abs() * (z.abs() <= ez) if act == "relu" else torch.zeros_like(z))
    if act:
        e = e + HB * (dz.abs() + e)
    out = [(y, ey + HB * (y.abs() + ey))]
    for ref, err, n, half in (
            (dz @ w, e @ w.abs() + (N + 2) * U * (dz.abs() @ w.abs()), N, HB),
            (dz.t() @ x, e.t() @ x.abs() + (M + 2) * U * (dz.abs().t() @ x.abs()), M,
             HB if w_type == BF16 else U),
            (dz.sum(0), e.sum(0) + (M + 2) * U * dz.abs().sum(0), M,
             HB if w_type == BF16 else U)):
        out.append((ref, err + half * (ref.abs() + err)))
    return out


def _inputs(M, N, K, bias, res, seed, w_type=BF16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(BF16)
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    b = torch.randn(N, generator=g).to(BF16) if bias else None
    r = torch.randn(M, N, generator=g).to(BF16) if res else None
    return x, w, b, r, torch.randn(M, N, generator=g).to(BF16)


def _check(got, ref, what):
    for name, x, (r, b) in zip(("y", "dx", "dw", "db"), got, ref):
        x = x.double().cpu()
        assert x.shape == r.shape and torch.isfinite(x).all(), f"{what} {name}"
        over = ((x - r).abs() - b).max().item() if x.numel() else 0.0
        assert over <= 0, f"{what} {name}: {over:.3e} over the bound"


def _case(dev, M, N, K, act, bias=True, res=True, seed=0, w_type=BF16):
    print(f"case M={M} N={N} K={K} {act} bias={bias} residual={res} {w_type}", flush=True)
    x, w, b, r, gy = _inputs(M, N, K, bias, res, seed)
    leaves = [x.to(dev).requires_grad_(), w.to(w_type).to(dev).requires_grad_()]
    leaves += [b.to(w_type).to(dev).requires_grad_()] if bias else []
    rd = r.to(dev).requires_grad_() if res else None
    y = linear_epilogue(leaves[0], leaves[1], leaves[2] if bias else None, activation=act,
                        residual=rd)
    grads = torch.autograd.grad(y, leaves + ([rd] if res else []), gy.to(dev))
    assert all(g.dtype == t.dtype for g, t in zip(grads, leaves))
    if res:
        assert torch.equal(grads[-1].cpu(), gy)
    _check([y.detach(), *grads[:len(leaves)]], _ref(x, w, b, r, gy, act, w_type), "linear")
    with torch.no_grad():
        alone = linear_epilogue(leaves[0], leaves[1], leaves[2] if bias else None, activation=act,
                                residual=rd)
    assert torch.equal(alone, y)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 768, 768), (5, 64, 100), (31, 47, 72), (33, 40, 65),
                                   (64, 8, 8), (130, 257, 200), (300, 96, 1000)])
def test_few_outputs(dev, M, N, K, act):
    _case(dev, M, N, K, act, seed=M + N)


@pytest.mark.parametrize("act,bias,res", [(None, True, True), ("relu", False, True),
                                          ("gelu", True, False), ("gelu", False, False)])
@pytest.mark.parametrize("M,N,K", [(1500, 1500, 64), (2100, 1024, 72), (2049, 1100, 99),
                                   (8200, 640, 128), (16500, 384, 40), (16385, 300, 65)])
def test_tiles(dev, M, N, K, act, bias, res):
    _case(dev, M, N, K, act, bias, res, seed=N)


@pytest.mark.parametrize("M,N,K", [(1100, 700, 96), (1001, 770, 99), (40, 5200, 264),
                                   (520, 1000, 1024)])
def test_between_few_outputs_and_tiles(dev, M, N, K):
    _case(dev, M, N, K, "gelu", seed=K)


# K of one stage, a part of one, and ends after each of the four buffers
@pytest.mark.parametrize("K", [8, 64, 72, 128, 192, 200, 256, 320, 456, 512])
def test_one_block_on_each_cu(dev, K):
    _case(dev, 1800, 1024, K, "gelu", seed=K)


@pytest.mark.parametrize("M,N,K", [(32700, 513, 1032), (32700, 513, 1025), (32641, 520, 1024)])
def test_many_tiles_of_a_long_contraction(dev, M, N, K):
    _case(dev, M, N, K, "relu", seed=N)


def test_fp32_parameters_and_inputs(dev):
    _case(dev, 700, 96, 160, "gelu", w_type=F32)
    x, w, b, r, gy = _inputs(50, 24, 40, True, True, 3)
    xf, rf = x.float().to(dev).requires_grad_(), r.float().to(dev).requires_grad_()
    y = linear_epilogue(xf, w.to(dev), b.to(dev), "relu", rf)
    dx, dr = torch.autograd.grad(y, (xf, rf), gy.to(dev))
    assert y.dtype == BF16 and dx.dtype == dr.dtype == F32
    _check([y, dx], _ref(x, w, b, r, gy, "relu"), "fp32 inputs")
    assert torch.equal(dr.cpu(), gy.float())


def test_shapes_strides_and_alignment(dev):
    x, w, b, r, _ = _inputs(60, 48, 64, True, True, 4)
    x, w, b, r = (t.to(dev) for t in (x, w, b, r))
    want = linear_epilogue(x, w, b, "gelu", r)
    three = linear_epilogue(x.view(3, 20, 64), w, b, "gelu", r.view(3, 20, 48))
    assert three.shape == (3, 20, 48) and torch.equal(three.view(60, 48), want)
    assert torch.equal(linear_epilogue(x[7], w, b, "gelu", r[7]), want[7])
    wide = torch.zeros(60, 200, dtype=BF16, device=dev)
    wide[:, 8:72] = x
    assert torch.equal(linear_epilogue(wide[:, 8:72], w, b, "gelu", r), want)
    odd = torch.empty(60 * 64 + 1, dtype=BF16, device=dev)[1:].view(60, 64)
    odd.copy_(x)
    assert torch.equal(linear_epilogue(odd, w, b, "gelu", r), want)
    assert torch.equal(linear_epilogue(x.t().contiguous().t(), w.t().contiguous().t(), b, "gelu",
                                       r.t().contiguous().t()), want)
    same = linear_epilogue(x[:1].expand(60, 64), w, b, "gelu", r[:1].expand(60, 48))
    assert torch.equal(same[3:4], want[:1])


@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_no_rows(dev, act):
    x = torch.empty(0, 16, dtype=BF16, device=dev, requires_grad=True)
    w = torch.ones(8, 16, dtype=BF16, device=dev, requires_grad=True)
    b = torch.ones(8, dtype=BF16, device=dev, requires_grad=True)
    y = linear_epilogue(x, w, b, act)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_only_some_gradients(dev):
    x, w, b, r, gy = (t.to(dev) for t in _inputs(40, 24, 32, True, True, 6))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    full = torch.autograd.grad(linear_epilogue(*leaves[:3], "gelu", leaves[3]), leaves, gy)
    for i, t in enumerate(leaves):
        args = [u if j == i else u.detach() for j, u in enumerate(leaves)]
        one, = torch.autograd.grad(linear_epilogue(*args[:3], "gelu", args[3]), t, gy)
        assert (one.float() - full[i].float()).abs().max() <= HB * full[i].float().abs().max()


def test_special_values_stay_in_their_row_and_column(dev):
    M, N, K = 2000, 1100, 64
    x = torch.ones(M, K, dtype=BF16, device=dev)
    w = torch.ones(N, K, dtype=BF16, device=dev)
    x[5, 3], x[1999, 63], w[1099, 0] = math.inf, math.nan, -math.inf
    y = linear_epilogue(x, w)
    ref = x.double() @ w.double().t()
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.isinf(), ref.isinf())
    for act, want in (("relu", torch.relu), ("gelu", torch.nn.functional.gelu)):
        v = torch.tensor([[math.inf], [-math.inf], [math.nan], [0.0], [-0.0], [300.0], [-300.0]],
                         dtype=BF16, device=dev)
        got = linear_epilogue(v, torch.ones(1, 1, dtype=BF16, device=dev), None, act)
        assert torch.equal(got.isnan(), want(v).isnan())
        assert torch.equal(got.nan_to_num(1.0, 2.0, 3.0), want(v).nan_to_num(1.0, 2.0, 3.0))


def test_the_same_bits_every_time_on_another_stream_and_captured(dev):
    x, w, b, r, gy = (t.to(dev) for t in _inputs(3000, 640, 256, True, True, 7))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def step():
        y = linear_epilogue(*leaves[:3], "gelu", leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    first = [t.clone() for t in step()]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(0.5)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(static, want))


def test_residual_may_be_the_output(dev):
    """The C entry with residual == y: each element is read before it is written."""
    x, w, b, r, _ = (t.to(dev) for t in _inputs(500, 72, 40, True, True, 8))
    want = linear_epilogue(x, w, b, "relu", r)
    y = r.clone()
    _lib.check(_lib.load().ngt_linear_fwd(x.data_ptr(), 40, w.data_ptr(), b.data_ptr(),
                                          y.data_ptr(), 500, 72, 40, ACTIVATIONS["relu"],
                                          y.data_ptr(), None, _lib.stream_ptr(dev)))
    assert torch.equal(y, want)


def test_refusals(dev):
    x = torch.zeros(4, 8, dtype=BF16, device=dev)
    w = torch.zeros(6, 8, dtype=BF16, device=dev)
    for args, err in (((x.cpu(), w), ValueError), ((x, w.cpu()), ValueError),
                      ((x.half(), w), TypeError), ((x, w[:, :7]), ValueError),
                      ((x, w, x[0]), ValueError), ((x, w, None, "tanh"), ValueError),
                      ((x, w, None, None, x), ValueError), ((x, w[:0]), ValueError),
                      ((x, w[0]), ValueError)):
        with pytest.raises(err):
            linear_epilogue(*args)
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(linear_epilogue(xg, w).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("w_type", [BF16, F32])
def test_the_cpp_node_and_the_python_class_give_the_same_bits(dev, act, w_type, monkeypatch):
    assert _lib.autograd_ext() is not None
    x, w, b, r, gy = (t.to(dev) for t in _inputs(300, 56, 104, True, True, 9))
    leaves = [t.requires_grad_() for t in (x.float(), w.to(w_type), b.to(w_type), r.float())]

    def step():
        y = linear_epilogue(leaves[0].view(3, 100, 104), *leaves[1:3], act,
                            leaves[3].view(3, 100, 56))
        return [y.detach(), *torch.autograd.grad(y, leaves, gy.view(3, 100, 56))]

    a = step()
    monkeypatch.setattr(_lib, "node_ext", lambda: None)
    assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(a, step()))
