"""norm_rotary against float64: results and gradients, each element within the bound of
the roundings made (oracle/rotary.py)."""
import math

import pytest
import torch

from neutrongt_amd import Rotary, _lib, norm_rotary
from oracle import rotary as OR

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _gain(d, g, dtype):
    return (1 + 0.2 * torch.randn(d, generator=g)).to(dtype)


def _case(dev, n, H, Hk, d, dim, layout, dtype, norm=(True, True), gain_dtype=F32, far=0, seed=0,
          pos_dtype=torch.int32, magnitude=1.0, joint=True, **kw):
    print(f"case n={n} H={H}/{Hk} d={d} dim={dim} {layout} {dtype} norm={norm} far={far}", flush=True)
    g = torch.Generator().manual_seed(seed)
    rot = Rotary(dim, layout=layout, magnitude=magnitude, device=dev, **kw) if dim else None
    pos = torch.randint(-far, far + 1, (n,), generator=g).to(pos_dtype) if dim else None
    xs, gains, gys = [], [], []
    for heads, with_norm in ((H, norm[0]), (Hk, norm[1])):
        if not heads:
            continue
        xs.append(torch.randn(n, heads, d, generator=g).to(dtype))
        gains.append(_gain(d, g, gain_dtype) if with_norm else None)
        gys.append(torch.randn(n, heads, d, generator=g).to(dtype))
    dev_x = [x.to(dev) for x in xs]
    if joint and Hk:
        both = torch.cat(dev_x, 1)
        dev_x = [both[:, :H].detach(), both[:, H:].detach()]
    leaves = [x.requires_grad_() for x in dev_x]
    dev_g = [t.to(dev).requires_grad_() if t is not None else None for t in gains]
    args = dict(positions=pos.to(dev) if dim else None, rotary=rot, q_gain=dev_g[0],
                k_gain=dev_g[1] if Hk else None, eps=1e-6)
    ys = norm_rotary(leaves[0], leaves[1] if Hk else None, **args)
    ys = ys if Hk else (ys,)
    wanted = leaves + [t for t in dev_g if t is not None]
    grads = list(torch.autograd.grad(ys, wanted, [t.to(dev) for t in gys]))
    with torch.no_grad():
        again = norm_rotary(leaves[0], leaves[1] if Hk else None, **args)
    assert all(torch.equal(a, b) for a, b in zip(again if Hk else (again,), ys))
    dgains = grads[len(leaves):]
    f = rot.frequencies if rot else None
    for i, (x, gain, gy) in enumerate(zip(xs, gains, gys)):
        ref = OR.bounds(x, gain, pos, f, layout, magnitude, 1e-6, gy, HALF[dtype], HALF[gain_dtype])
        got = [ys[i].detach(), grads[i], dgains.pop(0) if gain is not None else None]
        for name, t, r in zip(("y", "dx", "dgain"), got, ref):
            if r is None:
                continue
            assert t.dtype == (gain_dtype if name == "dgain" else dtype) and t.shape == r[0].shape
            over = ((t.double().cpu() - r[0]).abs() - r[1]).max().item() if t.numel() else 0.0
            assert over <= 0, f"{'qk'[i]} {name}: {over:.3e} over the bound"


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,Hk,d,dim", [(8, 8, 8, 8), (8, 2, 16, 16), (32, 32, 24, 24), (4, 1, 40, 20),
                                        (12, 12, 80, 80), (32, 8, 128, 128), (5, 5, 96, 24),
                                        (3, 1, 256, 64), (2, 2, 256, 256), (7, 3, 64, 32),
                                        (4, 4, 8, 2), (3, 3, 10, 6), (1, 1, 2, 2), (2, 1, 250, 10)])
def test_heads_and_layouts(dev, H, Hk, d, dim, layout, dtype):
    _case(dev, 37, H, Hk, d, dim, layout, dtype, far=5000, seed=d + dim)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 63, 257, 1500, 4099])
def test_rows(dev, n, dtype):
    _case(dev, n, 8, 2, 32, 32, "half", dtype, far=100, seed=n)


@pytest.mark.parametrize("H,Hk", [(700, 1), (1, 700), (300, 300)])
def test_many_heads(dev, H, Hk):
    _case(dev, 3, H, Hk, 6, 2, "half", F32, far=9, seed=H)
    _case(dev, 900, H, Hk, 8, 8, "half", BF16, far=9, seed=H)


@pytest.mark.parametrize("n", [9000, 20011])
def test_more_tiles_than_blocks_of_the_backward(dev, n):
    _case(dev, n, 4, 1, 16, 8, "interleaved", BF16, far=n, seed=n)


def test_more_rounds_of_many_heads(dev):
    _case(dev, 11003, 64, 64, 16, 16, "half", F32, far=11003, seed=8)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm", [(True, False), (False, True), (False, False)])
def test_norms_of_one_of_them_or_none(dev, norm, dtype):
    _case(dev, 130, 6, 2, 48, 48, "half", dtype, norm=norm, far=1000, seed=3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_alone_and_norm_alone(dev, dtype):
    _case(dev, 77, 6, 0, 64, 64, "half", dtype, far=10, seed=4)
    _case(dev, 77, 6, 2, 64, 0, "half", dtype, seed=5)
    _case(dev, 77, 6, 0, 64, 0, "half", dtype, norm=(True, False), seed=6)


def test_bf16_gains_and_int64_positions(dev):
    _case(dev, 200, 8, 4, 32, 32, "half", BF16, gain_dtype=BF16, far=1 << 20, seed=7,
          pos_dtype=torch.int64)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("far", [1 << 17, 1 << 28, (1 << 31) - 2])
def test_far_positions(dev, far, dtype):
    _case(dev, 60, 4, 4, 128, 128, "half", dtype, far=far, seed=8)
    _case(dev, 60, 4, 4, 64, 64, "interleaved", dtype, far=far, seed=9, scaling="linear", factor=8.0)


def test_scalings(dev):
    for kw in (dict(scaling="base", factor=4.0), dict(scaling="linear", factor=32.0),
               dict(scaling="parts", factor=16.0, trained_length=4096),
               dict(frequencies=torch.rand(32, dtype=torch.float64))):
        _case(dev, 64, 4, 2, 64, 64, "half", F32, far=60000, seed=10, magnitude=1.2, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_alignment(dev, dtype):
    g = torch.Generator().manual_seed(1)
    n, H, d = 50, 4, 32
    x = torch.randn(n, H, d, generator=g).to(dtype).to(dev)
    gy = torch.randn(n, H, d, generator=g).to(dtype).to(dev)
    gain = _gain(d, g, F32).to(dev)
    pos = torch.arange(n, device=dev)
    rot = Rotary(d, device=dev)
    want = norm_rotary(x, None, pos, rot, gain)
    leaf = x.clone().requires_grad_()
    want_dx, = torch.autograd.grad(norm_rotary(leaf, None, pos, rot, gain), leaf, gy)
    tol = HALF[dtype] * 4 * want.float().abs().max()

    def views(t):
        wide = torch.zeros(n, 3 * H, d, dtype=dtype, device=dev)
        wide[:, H:2 * H] = t
        yield wide[:, H:2 * H]                        # a part of a joint projection
        inner = torch.zeros(n, H, 3 * d, dtype=dtype, device=dev)
        inner[:, :, d:2 * d] = t
        yield inner[:, :, d:2 * d]                    # the parts side by side in each head
        odd = torch.zeros(n * H * d + 1, dtype=dtype, device=dev)[1:].view(n, H, d)
        odd.copy_(t)
        yield odd                                     # aligned to an element only
        yield t.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside
        yield t.transpose(1, 2).contiguous().transpose(1, 2)  # components outside

    for v, gv in zip(views(x), views(gy)):
        y = norm_rotary(v, None, pos, rot, gain)
        assert y.is_contiguous() and (y.float() - want.float()).abs().max() <= tol
        leaf = v.detach().requires_grad_()
        dx, = torch.autograd.grad(norm_rotary(leaf, None, pos, rot, gain), leaf, gv)
        assert (dx.float() - want_dx.float()).abs().max() <= HALF[dtype] * 4 * want_dx.float().abs().max()
    four = norm_rotary(x.view(5, 10, H, d), None, pos.view(5, 10), rot, gain)
    assert torch.equal(four.view(n, H, d), want)
    one = norm_rotary(x[3], None, pos[3], rot, gain)
    assert (one.float() - want[3].float()).abs().max() <= tol
    same = x[:1].expand(n, H, d).detach().requires_grad_()
    dx, = torch.autograd.grad(norm_rotary(same, None, pos, rot, gain), same,
                              gy[:1, :1, :1].expand(n, H, d))
    assert dx.shape == (n, H, d) and torch.isfinite(dx).all()


def test_offsets_behind_2_to_the_31(dev):
    """Rows whose offsets in elements pass 2^31, and rows 2^31 elements apart."""
    n, H, d = 5, 2, 8
    big = torch.empty((1 << 31) + 4096, dtype=BF16, device=dev)
    x = torch.randn(n, H, d, device=dev).to(BF16)
    pos, rot = torch.arange(n, device=dev), Rotary(d, device=dev)
    v = big.as_strided((n, H, d), ((1 << 29) + 16, d, 1))
    v.copy_(x)
    assert torch.equal(norm_rotary(v, None, pos, rot), norm_rotary(x, None, pos, rot))
    at = torch.as_strided(big, (n, H, d), (H * d, d, 1), (1 << 31) + 8)
    at.copy_(x)
    assert torch.equal(norm_rotary(at, None, pos, rot), norm_rotary(x, None, pos, rot))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_special_values_stay_in_their_head(dev, dtype):
    n, H, d, dim = 40, 6, 24, 16
    x = torch.randn(n, H, d, device=dev).to(dtype)
    gain, pos, rot = torch.ones(d, device=dev), torch.arange(n, device=dev), Rotary(dim, device=dev)
    clean = norm_rotary(x, None, pos, rot, gain)
    bad = x.clone()
    bad[3, 2, 5], bad[7, 0, 20], bad[9, 5, 0] = math.nan, math.inf, -math.inf
    y = norm_rotary(bad, None, pos, rot, gain)
    hit = torch.zeros(n, H, dtype=torch.bool, device=dev)
    hit[3, 2] = hit[7, 0] = hit[9, 5] = True
    assert torch.equal(y[~hit], clean[~hit]) and y[3, 2].isnan().all()
    # without a norm only the value's own pair, and an unturned one alone
    y, clean = norm_rotary(bad, None, pos, rot), norm_rotary(x, None, pos, rot)
    where = ~torch.isfinite(y)
    want = torch.zeros_like(where)
    want[3, 2, 5] = want[3, 2, 13] = want[7, 0, 20] = want[9, 5, 0] = want[9, 5, 8] = True
    assert torch.equal(where, want) and torch.equal(y[~want], clean[~want])
    zero = norm_rotary(torch.zeros_like(x), None, pos, rot, gain)
    assert not zero.any()


def test_only_some_gradients(dev):
    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn(60, h, 16, generator=g).to(BF16).to(dev) for h in (4, 2))
    gains = [_gain(16, g, F32).to(dev) for _ in range(2)]
    pos, rot = torch.arange(60, device=dev), Rotary(16, device=dev)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    leaves = [t.requires_grad_() for t in (q, k, *gains)]

    def run(args):
        return norm_rotary(args[0], args[1], pos, rot, args[2], args[3])

    full = torch.autograd.grad(run(leaves), leaves, (gq, gk))
    for i, t in enumerate(leaves):
        args = [u if j == i else u.detach() for j, u in enumerate(leaves)]
        one, = torch.autograd.grad([y for y in run(args) if y.requires_grad], t,
                                   [s for y, s in zip(run(args), (gq, gk)) if y.requires_grad])
        assert torch.equal(one, full[i])
    # one result's gradient alone: the other's is zero
    dq, dk, dgq, dgk = torch.autograd.grad(run(leaves)[0], leaves, gq, allow_unused=True)
    assert torch.equal(dq, full[0]) and not dk.any() and torch.equal(dgq, full[2]) and not dgk.any()


@pytest.mark.parametrize("node", [True, False])
def test_without_a_norm_the_input_is_not_kept(dev, node, monkeypatch):
    """What has no gain may change or go before the backward; what has one may not change."""
    if not node:
        monkeypatch.setattr(_lib, "node_ext", lambda: None)
    g = torch.Generator().manual_seed(4)
    q, k = (torch.randn(50, h, 16, generator=g).to(dev).requires_grad_() for h in (4, 2))
    gain, gq, gk = _gain(16, g, F32).to(dev), torch.randn_like(q), torch.randn_like(k)
    pos, rot = torch.arange(50, device=dev), Rotary(12, device=dev)
    for gains in ((None, None), (None, gain), (gain, None)):
        want = torch.autograd.grad(norm_rotary(q, k, pos, rot, *gains), (q, k), (gq, gk))
        ys = norm_rotary(q, k, pos, rot, *gains)
        with torch.no_grad():
            for t, gt in zip((q, k), gains):
                if gt is None:
                    t.add_(1)
        assert all(torch.equal(a, b) for a, b in
                   zip(torch.autograd.grad(ys, (q, k), (gq, gk)), want))
    ys = norm_rotary(q, k, pos, rot, gain)
    with torch.no_grad():
        q.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(ys, (q, k), (gq, gk))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rotate", [False, True])
def test_the_cpp_node_and_the_python_class_give_the_same_bits(dev, dtype, rotate, monkeypatch):
    assert _lib.autograd_ext() is not None
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(3, 70, h, 40, generator=g).to(dtype).to(dev).requires_grad_() for h in (6, 2))
    gains = [_gain(40, g, F32).to(dev).requires_grad_() for _ in range(2)]
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    pos = torch.arange(210, device=dev).view(3, 70) if rotate else None
    rot = Rotary(20, layout="interleaved", device=dev) if rotate else None

    def step():
        ys = norm_rotary(q, k, pos, rot, *gains)
        alone = norm_rotary(q, None, pos, rot)
        return [*(y.detach() for y in ys), alone.detach(),
                *torch.autograd.grad(ys, (q, k, *gains), (gq, gk))]

    a = step()
    monkeypatch.setattr(_lib, "node_ext", lambda: None)
    assert all(torch.equal(p, r) and p.dtype == r.dtype and p.shape == r.shape
               for p, r in zip(a, step()))


def test_the_same_bits_every_time_on_another_stream_and_captured(dev):
    g = torch.Generator().manual_seed(11)
    q, k = (torch.randn(3000, h, 64, generator=g).to(BF16).to(dev).requires_grad_() for h in (8, 2))
    gains = [_gain(64, g, F32).to(dev).requires_grad_() for _ in range(2)]
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    pos, rot = torch.arange(3000, device=dev), Rotary(64, device=dev)

    def step():
        ys = norm_rotary(q, k, pos, rot, *gains)
        return [*(y.detach() for y in ys), *torch.autograd.grad(ys, (q, k, *gains), (gq, gk))]

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
            q.mul_(0.5)
            pos.add_(7)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(static, want))


def test_refusals(dev):
    q, k = torch.zeros(4, 8, 16, device=dev), torch.zeros(4, 2, 16, device=dev)
    pos, rot, gain = torch.arange(4, device=dev), Rotary(16, device=dev), torch.ones(16, device=dev)
    for args, kw, err in (((q.cpu(),), {}, ValueError), ((q.half(),), {}, TypeError),
                          ((q, k.to(BF16)), {}, TypeError), ((q, k[:3]), {}, ValueError),
                          ((q, k, pos), {}, ValueError), ((q, k, None, rot), {}, ValueError),
                          ((q, k, pos, "rotary"), {}, TypeError),
                          ((q, k, pos.float(), rot), {}, ValueError),
                          ((q, k, pos[:3], rot), {}, ValueError),
                          ((q, k, pos.cpu(), rot), {}, ValueError),
                          ((q, k, pos, Rotary(18, device=dev)), {}, ValueError),
                          ((q, k, pos, rot, gain[:8]), {}, ValueError),
                          ((q, k, pos, rot, gain.double()), {}, ValueError),
                          ((q, k, pos, rot, gain.to(BF16)), {}, ValueError),
                          ((q, None, pos, rot, gain, gain), {}, ValueError),
                          ((q[..., :15],), {}, ValueError), ((q[:, :0],), {}, ValueError),
                          ((torch.zeros(2, 1, 258, device=dev),), {}, ValueError),
                          ((q, k, pos, rot), dict(eps=-1.0), ValueError),
                          ((q, k, pos, rot), dict(eps=math.nan), ValueError)):
        with pytest.raises(err):
            norm_rotary(*args, **kw)
    qg = q.clone().requires_grad_()
    g, = torch.autograd.grad(norm_rotary(qg, None, pos, rot, gain).sum(), qg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
