"""gated_linear against float64: y = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients,
each element within the bound of the roundings made.

The products of bf16 values are exact in fp32 (u = 2^-24 its half step, h = 2^-8
bf16's), a sum of n of them is off by at most n u of their absolute values.
  z:     e = (K + 2) u (sum|x||w| + |b|), for zg and zu
  a:     act(zg): 1.13 e_g (no slope is larger) + 8 u (|zg| + |a|)
  slope: act'(zg): 0.8 e_g (no second derivative is larger) + 16 u (1 + |zg|); relu's may
         differ where |zg| <= e_g
  y:     |zu| e_a + (|a| + e_a) e_u + 2 u |y|, then h |y|
  kept:  zu slope and a, the same way, each rounded to 12 bits of mantissa, off by at
         most k = 2^-12 of itself; dz = dy times them, rounded to bf16
  dx, dw, db: sums of dz's error and n u of the terms, then h (bf16) or nothing"""
import math

import pytest
import torch

from neutrongt_amd import _lib, gated_linear
from neutrongt_amd.linear import GATES

pytestmark = pytest.mark.gpu
U, HB, HK = 2.0 ** -24, 2.0 ** -8, 2.0 ** -12
BF16, F32 = torch.bfloat16, torch.float32


def _act(z, act):
    """act(z), act'(z)."""
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def _ref(x, wg, wu, bg, bu, gy, act, w_type=BF16):
    """[(value, bound)] of y, dx, dwg, dwu, dbg, dbu."""
    x, wg, wu, gy = (t.double() for t in (x, wg, wu, gy))
    (M, K), N = x.shape, wg.shape[0]
    none = torch.zeros(N, dtype=torch.float64)
    bg, bu = (b.double() if b is not None else none for b in (bg, bu))
    zg, zu = x @ wg.t() + bg, x @ wu.t() + bu
    eg, eu = ((K + 2) * U * (x.abs() @ w.abs().t() + b.abs()) for w, b in ((wg, bg), (wu, bu)))
    a, s = _act(zg, act)
    ea = 1.13 * eg + 8 * U * (zg.abs() + a.abs())
    es = ((zg.abs() <= eg).double() if act == "relu" else
          0.8 * eg + 16 * U * (1 + zg.abs()) if act else torch.zeros_like(zg))
    up = lambda v, e, half=HB: e + half * (v.abs() + e)
    y = a * zu
    ey = zu.abs() * ea + (a.abs() + ea) * eu + 2 * U * y.abs()
    out = [(y, up(y, ey))]
    kg = zu * s
    ekg = up(kg, zu.abs() * es + (s.abs() + es) * eu + 2 * U * kg.abs(), HK)
    dzs = [(gy * v, up(gy * v, gy.abs() * e)) for v, e in ((kg, ekg), (a, up(a, ea, HK)))]
    dx = dzs[0][0] @ wg + dzs[1][0] @ wu
    e = sum(ez @ w.abs() + (2 * N + 2) * U * (z.abs() @ w.abs())
            for (z, ez), w in zip(dzs, (wg, wu)))
    out.append((dx, up(dx, e)))
    half = HB if w_type == BF16 else U
    for dim in (0, 1):
        for z, ez in dzs:
            v, e = ((z.t() @ x, ez.t() @ x.abs() + (M + 2) * U * (z.abs().t() @ x.abs())) if dim == 0
                    else (z.sum(0), ez.sum(0) + (M + 2) * U * z.abs().sum(0)))
            out.append((v, e + half * (v.abs() + e)))
    return out


def _inputs(M, N, K, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(BF16)
    wg, wu = ((torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16) for _ in range(2))
    bg, bu = (torch.randn(N, generator=g).to(BF16) if bias else None for _ in range(2))
    return x, wg, wu, bg, bu, torch.randn(M, N, generator=g).to(BF16)


NAMES = ("y", "dx", "dwg", "dwu", "dbg", "dbu")


def _check(got, ref, what):
    for name, x, (r, b) in zip(NAMES, got, ref):
        x = x.double().cpu()
        assert x.shape == r.shape and torch.isfinite(x).all(), f"{what} {name}"
        over = ((x - r).abs() - b).max().item() if x.numel() else 0.0
        assert over <= 0, f"{what} {name}: {over:.3e} over the bound"


def _case(dev, M, N, K, act, bias=True, seed=0, w_type=BF16):
    print(f"case M={M} N={N} K={K} {act} bias={bias} {w_type}", flush=True)
    x, wg, wu, bg, bu, gy = _inputs(M, N, K, bias, seed)
    leaves = [x.to(dev).requires_grad_()]
    leaves += [t.to(w_type).to(dev).requires_grad_() for t in (wg, wu, bg, bu) if t is not None]
    y = gated_linear(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, gy.to(dev))
    assert y.dtype == BF16 and all(g.dtype == t.dtype for g, t in zip(grads, leaves))
    _check([y.detach(), *grads], _ref(x, wg, wu, bg, bu, gy, act, w_type), "gated")
    with torch.no_grad():
        assert torch.equal(gated_linear(*leaves, activation=act), y)


@pytest.mark.parametrize("act", list(GATES))
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 768, 768), (5, 64, 100), (16, 48, 256), (17, 40, 264),
                                   (31, 47, 72), (33, 40, 65), (64, 8, 8), (130, 257, 200),
                                   (300, 96, 1000)])
def test_small(dev, M, N, K, act):
    _case(dev, M, N, K, act, seed=M + N)


@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True), ("relu", False)])
@pytest.mark.parametrize("M,N,K", [(1500, 1500, 64), (2100, 1024, 72), (2049, 1100, 99),
                                   (8200, 640, 128), (16500, 384, 40), (16385, 300, 65),
                                   (520, 1000, 1024), (40, 5200, 264), (257, 513, 520)])
def test_tiles(dev, M, N, K, act, bias):
    _case(dev, M, N, K, act, bias, seed=N)


@pytest.mark.parametrize("M,N,K", [(512, 72, 136), (513, 264, 520), (600, 8, 8), (5000, 136, 264),
                                   (511, 264, 520), (70000, 40, 24), (777, 1000, 1288),
                                   (3001, 513, 264), (2000, 264, 1031), (1025, 769, 769), (70001, 41, 23),
                                   (900, 1001, 3), (64, 7, 2049)])
def test_gradients_of_whole_pieces_with_edges(dev, M, N, K):
    _case(dev, M, N, K, "silu", seed=M)


# a long contraction of the forward for few blocks, cut into several and not
@pytest.mark.parametrize("M,N,K", [(1, 64, 8192), (16, 16, 4096), (33, 256, 4104), (64, 40, 5000),
                                   (5, 33, 8191), (65, 64, 8192), (200, 256, 4096), (300, 136, 2056),
                                   (70, 61, 4097), (130, 257, 3001), (64, 1024, 2048), (449, 520, 1992)])
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True)])
def test_few_blocks_and_long_contractions(dev, M, N, K, act, bias):
    _case(dev, M, N, K, act, bias, seed=K)


# a contraction over many outputs for few blocks, cut into several and not
@pytest.mark.parametrize("M,N,K", [(1, 1024, 520), (33, 2048, 512), (64, 4096, 8), (65, 1000, 1288),
                                   (200, 256, 264), (300, 1288, 72), (71, 1001, 33), (130, 2050, 65),
                                   (450, 520, 2048)])
@pytest.mark.parametrize("w_type", [BF16, F32])
def test_gradients_of_few_rows_and_many_outputs(dev, M, N, K, w_type):
    _case(dev, M, N, K, "silu", bias=True, w_type=w_type, seed=N)


# a stage of the contraction, a part of one, several
@pytest.mark.parametrize("K", [8, 56, 64, 72, 128, 192, 200, 256, 320, 456, 512])
def test_lengths_of_the_contraction(dev, K):
    _case(dev, 1800, 1024, K, "silu", seed=K)


def test_fp32_parameters_and_inputs(dev):
    _case(dev, 700, 96, 160, "silu", w_type=F32)
    x, wg, wu, _, _, gy = _inputs(50, 24, 40, False, 3)
    xf = x.float().to(dev).requires_grad_()
    y = gated_linear(xf, wg.to(dev), wu.to(dev), activation="gelu")
    dx, = torch.autograd.grad(y, xf, gy.to(dev))
    assert y.dtype == BF16 and dx.dtype == F32
    _check([y, dx], _ref(x, wg, wu, None, None, gy, "gelu"), "fp32 inputs")


def test_shapes_strides_and_alignment(dev):
    x, wg, wu, bg, bu, _ = (t.to(dev) for t in _inputs(60, 48, 64, True, 4))
    want = gated_linear(x, wg, wu, bg, bu)
    three = gated_linear(x.view(3, 20, 64), wg, wu, bg, bu)
    assert three.shape == (3, 20, 48) and torch.equal(three.view(60, 48), want)
    tol = 4 * HB * want.float().abs().max()
    assert (gated_linear(x[7], wg, wu, bg, bu).float() - want[7].float()).abs().max() <= tol
    wide = torch.zeros(60, 200, dtype=BF16, device=dev)
    wide[:, 8:72] = x
    joint = torch.cat([wg, wu])
    odd = torch.empty(60 * 64 + 1, dtype=BF16, device=dev)[1:].view(60, 64)
    odd.copy_(x)
    for v, a, b in ((wide[:, 8:72], joint[:48], joint[48:]), (odd, wg, wu),
                    (x.t().contiguous().t(), wg.t().contiguous().t(), wu)):
        assert (gated_linear(v, a, b, bg, bu).float() - want.float()).abs().max() <= tol
    # the backward of weights and rows that are not aligned, in the tiled form too
    for m in (60, 600):
        x, wg, wu, _, _, gy = _inputs(m, 72, 64, False, m)
        odd = [torch.empty(t.numel() + 1, dtype=BF16, device=dev)[1:].view(t.shape) for t in (x, wg, wu, gy)]
        for o, t in zip(odd, (x, wg, wu, gy)):
            o.copy_(t)
        leaves = [t.requires_grad_() for t in odd[:3]]
        y = gated_linear(*leaves)
        _check([y.detach(), *torch.autograd.grad(y, leaves, odd[3])],
               _ref(x, wg, wu, None, None, gy, "silu"), "odd")
    x, wg, wu, bg, bu, _ = (t.to(dev) for t in _inputs(60, 48, 64, True, 4))
    same = gated_linear(x[:1].expand(60, 64), wg, wu, bg, bu)
    assert (same[3].float() - want[0].float()).abs().max() <= tol


@pytest.mark.parametrize("act", list(GATES))
def test_no_rows(dev, act):
    x = torch.empty(0, 16, dtype=BF16, device=dev, requires_grad=True)
    ps = [torch.ones(s, dtype=BF16, device=dev, requires_grad=True) for s in ((8, 16), (8, 16), 8, 8)]
    y = gated_linear(x, *ps, activation=act)
    dx, *gs = torch.autograd.grad(y, (x, *ps), torch.empty_like(y))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not any(g.any() for g in gs)


@pytest.mark.parametrize("N", [32768, 32767])
def test_offsets_behind_2_to_the_31(dev, N):
    """70,000 rows: the last rows' results, and the last outputs' weights' gradients."""
    M, K = 70000, 16
    x, (_, wg, wu, *_) = _inputs(M, 1, K, False, 1)[0], _inputs(1, N, K, False, 2)
    g = torch.Generator(device=dev).manual_seed(2)
    gy = torch.randn(M, N, dtype=BF16, device=dev, generator=g)
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu)]
    y = gated_linear(*leaves)
    dx, dg, du = torch.autograd.grad(y, leaves, gy)
    ref = _ref(x[-3:], wg, wu, None, None, gy[-3:].cpu(), "silu")
    _check([y[-3:].detach(), dx[-3:]], ref[:2], "last rows")
    ref = _ref(x, wg[-2:], wu[-2:], None, None, gy[:, -2:].cpu(), "silu")
    _check([dg[-2:], du[-2:]], ref[2:4], "last outputs")


def test_only_some_gradients_and_one_bias(dev):
    x, wg, wu, bg, bu, gy = (t.to(dev) for t in _inputs(40, 24, 32, True, 6))
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    full = torch.autograd.grad(gated_linear(*leaves), leaves, gy)
    for i, t in enumerate(leaves):
        args = [u if j == i else u.detach() for j, u in enumerate(leaves)]
        one, = torch.autograd.grad(gated_linear(*args), t, gy)
        assert (one.float() - full[i].float()).abs().max() <= HB * full[i].float().abs().max()
    for b in (dict(b_gate=leaves[3]), dict(b_up=leaves[4])):
        bias, = b.values()
        y = gated_linear(x, wg, wu, **b)
        got = torch.autograd.grad(y, (x, wg, wu, bias), gy)
        cpu = [t.detach().cpu() for t in (x, wg, wu)]
        pair = [b[n].detach().cpu() if n in b else None for n in ("b_gate", "b_up")]
        ref = _ref(*cpu, *pair, gy.cpu(), "silu")
        _check([y.detach(), *got[:3]], ref, "one bias")
        _check([got[3]], [ref[4 if "b_gate" in b else 5]], "its gradient")


def test_the_same_tensor_twice(dev):
    """Both layers from one weight: its gradient is the sum of both."""
    x, w, _, b, _, gy = (t.to(dev) for t in _inputs(100, 40, 48, True, 8))
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    dw, db = torch.autograd.grad(gated_linear(x, w, w, b, b), (w, b), gy)
    parts = [t.detach().clone().requires_grad_() for t in (w, w, b, b)]
    g = torch.autograd.grad(gated_linear(x, *parts), parts, gy)
    assert torch.equal(dw, g[0] + g[1]) and torch.equal(db, g[2] + g[3])


def test_special_values_stay_in_their_row_and_column(dev):
    M, N, K = 2000, 1100, 64
    x, wg, wu = (torch.ones(s, dtype=BF16, device=dev) for s in ((M, K), (N, K), (N, K)))
    x[5, 3], x[1999, 63], wg[1099, 0], wu[7, 1] = math.inf, math.nan, -math.inf, math.nan
    y = gated_linear(x, wg, wu, activation=None)
    ref = (x.double() @ wg.double().t()) * (x.double() @ wu.double().t())
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.isinf(), ref.isinf())
    v = torch.tensor([[math.inf], [-math.inf], [math.nan], [0.0], [-0.0], [300.0], [-300.0]],
                     dtype=BF16, device=dev)
    one = torch.ones(1, 1, dtype=BF16, device=dev)
    zero, bias = torch.zeros_like(one), torch.ones(1, dtype=BF16, device=dev)
    for act, f in (("relu", torch.relu), ("gelu", torch.nn.functional.gelu),
                   ("silu", torch.nn.functional.silu)):
        # the gate's own value: the other product is zero for finite rows, its bias 1
        got = gated_linear(v, one, zero, None, bias, activation=act)
        want = f(v.double()).to(BF16) * (v * 0 + 1)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(1.0, 2.0, 3.0) + 0, want.nan_to_num(1.0, 2.0, 3.0) + 0)


@pytest.mark.parametrize("M,N,K", [(3000, 640, 256), (20, 640, 256), (70, 61, 33), (40, 64, 4096),
                                   (100, 33, 2049), (600, 513, 520)])
def test_the_same_bits_every_time_on_another_stream_and_captured(dev, M, N, K):
    x, wg, wu, bg, bu, gy = (t.to(dev) for t in _inputs(M, N, K, True, 7))
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]

    def step():
        y = gated_linear(*leaves)
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
    for _ in range(3):
        with torch.no_grad():
            x.mul_(0.5)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(static, want))


def test_refusals(dev):
    x = torch.zeros(4, 8, dtype=BF16, device=dev)
    w = torch.zeros(6, 8, dtype=BF16, device=dev)
    b = torch.zeros(6, dtype=BF16, device=dev)
    for args, err in (((x.cpu(), w, w), ValueError), ((x, w.cpu(), w), ValueError),
                      ((x, w, w.cpu()), ValueError), ((x.half(), w, w), TypeError),
                      ((x, w, w.double()), TypeError), ((x, w[:, :7], w[:, :7]), ValueError),
                      ((x, w, w[:5]), ValueError), ((x, w, w, x[0]), ValueError),
                      ((x, w, w, b, x[0]), ValueError), ((x, w, w, None, None, "tanh"), ValueError),
                      ((x, w[:0], w[:0]), ValueError), ((x, w[0], w[0]), ValueError)):
        with pytest.raises(err):
            gated_linear(*args)
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(gated_linear(xg, w, w).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("act", list(GATES))
@pytest.mark.parametrize("w_type", [BF16, F32])
def test_the_cpp_node_and_the_python_class_give_the_same_bits(dev, act, w_type, monkeypatch):
    assert _lib.autograd_ext() is not None
    x, wg, wu, bg, bu, gy = (t.to(dev) for t in _inputs(300, 56, 104, True, 9))
    leaves = [t.requires_grad_() for t in (x.float(), *(t.to(w_type) for t in (wg, wu, bg, bu)))]

    def step():
        y = gated_linear(leaves[0].view(3, 100, 104), *leaves[1:], activation=act)
        return [y.detach(), *torch.autograd.grad(y, leaves, gy.view(3, 100, 56))]

    a = step()
    monkeypatch.setattr(_lib, "node_ext", lambda: None)
    assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(a, step()))
