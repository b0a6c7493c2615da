"""Attention over packed windows against the float64 oracle: out, dQ, dK, dV and
the bias table's gradient, each element within the bound that oracle.packed.bounds
derives from the roundings made."""
import math

import pytest
import torch

from neutrongt_amd import PackedWindows, _lib, packed_attention
from oracle import packed as OP

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def _inputs(ql, kl, H, hkv, d, dtype, buckets=0, seed=0, cut=0.05):
    g = torch.Generator().manual_seed(seed)
    q, go = (torch.randn(sum(ql), H, d, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(sum(kl), hkv, d, generator=g).to(dtype) for _ in range(2))
    table = ids = None
    if buckets:
        n = sum(a * b for a, b in zip(ql, kl))
        table = torch.randn(buckets, H, generator=g).to(dtype)
        ids = torch.randint(0, buckets, (n,), generator=g)
        ids[torch.rand(n, generator=g) < cut] = 255
    return q, k, v, go, table, ids


def _run(dev, q, k, v, go, table, ids, win, scale=None):
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    more = {}
    if table is not None:
        leaves.append(table.to(dev).requires_grad_())
        more = dict(bias_table=leaves[3], buckets=win.pack_buckets(ids.to(dev)))
    out = packed_attention(*leaves[:3], win, scale=scale, **more)
    return [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]


def _check(got, ref, bound, what):
    for name, x, r, b in zip(("out", "dq", "dk", "dv", "dtable"), got, ref, bound):
        x = x.double().cpu()
        assert x.shape == r.shape, f"{what} {name}"
        assert torch.isfinite(x).all(), f"{what} {name}: not finite"
        over = ((x - r).abs() - b).max().item() if x.numel() else 0.0
        assert over <= 0, f"{what} {name}: {over:.3e} over the bound"


def _case(dev, ql, kl, H, hkv, d, dtype, causal=False, buckets=0, seed=0, scale=None):
    print(f"case {ql} {kl} H={H}/{hkv} d={d} {dtype} causal={causal} buckets={buckets}", flush=True)
    q, k, v, go, table, ids = _inputs(ql, kl, H, hkv, d, dtype, buckets, seed)
    win = PackedWindows(ql, kl, causal=causal, device=dev)
    got = _run(dev, q, k, v, go, table, ids, win, scale)
    ref, bound = OP.bounds(q, k, v, go, ql, kl, HALF[dtype], causal, scale, table, ids)
    _check(got, ref, bound, "packed")
    with torch.no_grad():  # the same forward without what the backward needs
        more = {} if table is None else dict(bias_table=table.to(dev),
                                             buckets=win.pack_buckets(ids.to(dev)))
        alone = packed_attention(q.to(dev), k.to(dev), v.to(dev), win, scale=scale, **more)
    assert torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 128])
def test_head_sizes(dev, dtype, d):
    _case(dev, [33, 70, 1], [33, 70, 1], 2, 2, d, dtype, causal=d in (16, 40, 128), seed=d)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [
    ([1], [1]), ([0, 1, 0], [0, 1, 0]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [63, 64, 65]),
    ([127, 128, 129, 0, 5], [127, 128, 129, 0, 5]), ([5, 40, 3], [200, 17, 64]),
    ([9, 0, 2, 70], [0, 9, 1, 5]), ([200], [130])])
def test_lengths(dev, dtype, causal, lengths):
    _case(dev, *lengths, 4, 2, 16, dtype, causal=causal, seed=sum(lengths[0]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", [(1, 1), (6, 3), (8, 1), (12, 4), (16, 8)])
def test_grouped_heads(dev, dtype, heads):
    _case(dev, [40, 90], [70, 90], *heads, 32, dtype, causal=True, seed=heads[0])


@pytest.mark.parametrize("dtype,d", [(F32, 16), (BF16, 16), (BF16, 64), (BF16, 128), (F32, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_blocks_of_four_waves(dev, dtype, d, causal):
    """Enough rows and heads for 128-row blocks."""
    _case(dev, [700, 300, 150], [700, 350, 150], 64, 64 if d == 16 else 32, d, dtype,
          causal=causal, seed=7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,keys", [([1, 1, 1], [129, 1, 2000]), ([4, 0, 1, 2], [700, 50, 0, 33]),
                                       ([8, 8], [3000, 5]), ([1] * 9, [160] * 9)])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_a_few_rows_per_window(dev, dtype, rows, keys, d):
    _case(dev, rows, keys, 8, 2, d, dtype, causal=True, seed=d)
    _case(dev, rows, keys, 4, 4, d, dtype, causal=False, seed=d + 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,H,hkv,d,buckets,causal", [
    (([70, 3, 30], [70, 3, 30]), 4, 4, 8, 7, False), (([65, 129], [65, 129]), 8, 8, 24, 64, False),
    (([50, 20], [130, 20]), 6, 2, 64, 65, True), (([100, 1], [100, 1]), 2, 2, 128, 255, False),
    (([40, 40], [40, 40]), 4, 2, 40, 1, True), (([1, 2, 1], [300, 140, 1]), 8, 2, 32, 31, False),
    (([1, 1], [4000, 130]), 8, 8, 64, 12, True), (([400, 100], [400, 130]), 64, 64, 16, 40, True),
    (([300], [300]), 64, 64, 16, 200, False)])
def test_bias(dev, dtype, lengths, H, hkv, d, buckets, causal):
    _case(dev, *lengths, H, hkv, d, dtype, causal=causal, buckets=buckets, seed=buckets)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [([60, 35], [60, 35]), ([1, 2], [200, 64])])
def test_masks_that_leave_rows_empty(dev, dtype, lengths):
    ql, kl = lengths
    q, k, v, go, table, ids = _inputs(ql, kl, 4, 4, 16, dtype, 9, seed=3)
    first = ids[:ql[0] * kl[0]].view(ql[0], kl[0])
    first[0] = 255            # not attended
    first[-1] = -3            # below the table
    first[:, kl[0] // 2:] = 9  # the first id behind it
    table[4] = -math.inf      # a bucket that never counts
    second = ids[ql[0] * kl[0]:].view(ql[1], kl[1])
    second[0] = 4             # a row of nothing but that bucket
    win = PackedWindows(ql, kl, device=dev)
    got = _run(dev, q, k, v, go, table, ids, win)
    seen = torch.where(ids == 4, 255, ids)  # the oracle takes the bucket out
    table0 = table.clone()
    table0[4] = 0
    ref, bound = OP.bounds(q, k, v, go, ql, kl, HALF[dtype], False, None, table0, seen)
    _check(got, ref, bound, "empty rows")
    assert got[0][0].abs().max() == 0 and got[0][ql[0]].abs().max() == 0
    assert got[4][4].abs().max() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_of_the_types_lowest_value_is_attended(dev, dtype):
    ql = [40, 20]
    q, k, v, go, table, ids = _inputs(ql, ql, 2, 2, 16, dtype, 5, seed=4, cut=0.0)
    table[2] = torch.finfo(dtype).min
    ids[:40 * 40].view(40, 40)[3] = 2  # nothing greater: equal weights
    out = packed_attention(q.to(dev), k.to(dev), v.to(dev), win := PackedWindows(ql, device=dev),
                           bias_table=table.to(dev), buckets=win.pack_buckets(ids.to(dev)))
    mean = v[:40].double().mean(0)
    half = HALF[dtype]
    bound = (half + 64 * 2.0 ** -24) * v[:40].double().abs().mean(0) + half * mean.abs()
    assert ((out[3].double().cpu() - mean).abs() <= bound * 1.01).all()
    assert torch.isfinite(out).all()


def test_another_windows_nan_and_inf_stay_there(dev):
    for dtype in (F32, BF16):
        ql = [37, 50, 3]
        q, k, v, go, _, _ = _inputs(ql, ql, 2, 2, 32, dtype, seed=5)
        win = PackedWindows(ql, device=dev)
        want = _run(dev, q, k, v, go, None, None, win)
        for t in (q, k, v, go):
            t[37:87] = math.nan
            t[40] = math.inf
        got = _run(dev, q, k, v, go, None, None, win)
        for a, b in zip(got, want):
            assert torch.equal(a[:37], b[:37]) and torch.equal(a[87:], b[87:])


def test_views_of_a_joint_projection_and_other_strides(dev):
    ql = [45, 80]
    n, H, d = sum(ql), 4, 24
    for dtype in (F32, BF16):
        win = PackedWindows(ql, causal=True, device=dev)
        g = torch.Generator().manual_seed(6)
        joint = torch.randn(n, 3, H, d, generator=g).to(dtype).to(dev)
        want = packed_attention(*(joint[:, i].contiguous() for i in range(3)), win)
        assert torch.equal(packed_attention(*joint.unbind(1), win), want)
        heads_first = [joint[:, i].transpose(0, 1).contiguous().transpose(0, 1) for i in range(3)]
        assert torch.equal(packed_attention(*heads_first, win), want)
        odd = torch.empty(n * H * d + 1, dtype=dtype, device=dev)[1:].view(n, H, d)
        odd.copy_(joint[:, 0])
        assert torch.equal(packed_attention(odd, joint[:, 1], joint[:, 2], win), want)
        wide = joint[:1, 1].expand(n, H, d)  # one row for all: stride 0
        same = packed_attention(joint[:, 0], wide, joint[:, 2], win)
        assert torch.equal(same, packed_attention(joint[:, 0], wide.contiguous(), joint[:, 2], win))


def test_gradient_of_a_broadcast_input_and_of_a_strided_output_gradient(dev):
    ql, H, d = [30, 34], 2, 16
    q, k, v, go, _, _ = _inputs(ql, ql, H, H, d, F32, seed=8)
    win = PackedWindows(ql, device=dev)
    one = v[:1].to(dev).requires_grad_()
    got, = torch.autograd.grad(
        packed_attention(q.to(dev), k.to(dev), one.expand(64, H, d), win), one, go.to(dev))
    ref, bound = OP.bounds(q, k, v[:1].expand(64, H, d), go, ql, ql, HALF[F32])
    err = (got.double().cpu() - ref[3].sum(0, keepdim=True)).abs()
    assert (err <= bound[3].sum(0, keepdim=True) + 64 * 2.0 ** -24 * ref[3].abs().sum(0)).all()
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    gt = go.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    a = torch.autograd.grad(packed_attention(*leaves, win), leaves, gt)
    b = torch.autograd.grad(packed_attention(*leaves, win), leaves, go.to(dev))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_only_some_inputs_want_gradients(dev):
    ql = [33, 20]
    q, k, v, go, table, ids = _inputs(ql, ql, 2, 2, 16, BF16, 6, seed=9)
    win = PackedWindows(ql, device=dev)
    full = _run(dev, q, k, v, go, table, ids, win)
    b = win.pack_buckets(ids.to(dev))
    t = table.to(dev).requires_grad_()
    out = packed_attention(q.to(dev), k.to(dev), v.to(dev), win, bias_table=t, buckets=b)
    assert torch.equal(torch.autograd.grad(out, t, go.to(dev))[0], full[4])
    kk = k.to(dev).requires_grad_()
    out = packed_attention(q.to(dev), kk, v.to(dev), win, bias_table=table.to(dev), buckets=b)
    assert torch.equal(torch.autograd.grad(out, kk, go.to(dev))[0], full[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_every_time_and_on_another_stream(dev, dtype):
    ql = [150, 300, 7]
    q, k, v, go, table, ids = _inputs(ql, ql, 8, 4, 32, dtype, 20, seed=10)
    win = PackedWindows(ql, causal=True, device=dev)
    a = _run(dev, q, k, v, go, table, ids, win)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        b = _run(dev, q, k, v, go, table, ids, win)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_pack_buckets_layouts_and_id_types(dev):
    ql, kl = [70, 0, 5, 64], [33, 4, 130, 0]
    win = PackedWindows(ql, kl, device=dev)
    g = torch.Generator().manual_seed(11)
    mats = [torch.randint(-2, 300, (a, b), generator=g) for a, b in zip(ql, kl)]
    flat = torch.cat([m.flatten() for m in mats])
    want_q, want_k = [], []
    up = lambda n: (n + 63) // 64 * 64
    for m in mats:
        m = torch.where((m < 0) | (m > 255), 255, m).to(torch.uint8)
        a, b = m.shape
        by_q = torch.full((a, up(b)), 255, dtype=torch.uint8)
        by_q[:, :b] = m
        by_k = torch.full((b, up(a)), 255, dtype=torch.uint8)
        by_k[:, :a] = m.t()
        want_q.append(by_q.flatten())
        want_k.append(by_k.flatten())
    for ids in (flat, flat.int(), flat.short(), [m.to(dev) for m in mats]):
        b = win.pack_buckets(ids if isinstance(ids, list) else ids.to(dev))
        assert torch.equal(b.by_query.cpu(), torch.cat(want_q))
        assert torch.equal(b.by_key.cpu(), torch.cat(want_k))
    small = flat.clamp(0, 255).to(torch.uint8)
    b = win.pack_buckets(small.to(dev))
    assert torch.equal(b.by_query.cpu()[:70 * 64].view(70, 64)[:, :33],
                       small[:70 * 33].view(70, 33))


def test_captured_step_replays_with_new_inputs(dev):
    """Forward and backward in one graph, replayed with other inputs and other
    eager work in between; every replay against the eager bits."""
    ql = [90, 40, 1]
    win = PackedWindows(ql, causal=False, device=dev)
    sets = [_inputs(ql, ql, 4, 2, 32, BF16, 12, seed=s) for s in (20, 21, 22)]
    b = win.pack_buckets(sets[0][5].to(dev))
    cur = [t.to(dev) for t in sets[0][:5]]
    leaves = [cur[i].requires_grad_() for i in (0, 1, 2, 4)]

    def step():
        out = packed_attention(*leaves[:3], win, bias_table=leaves[3], buckets=b)
        return [out.detach(), *torch.autograd.grad(out, leaves, cur[3])]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for s in (1, 2, 0, 1):
        with torch.no_grad():
            for t, x in zip(cur, sets[s][:5]):
                t.copy_(x)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(static, want))


def test_captured_serving_step(dev):
    win = PackedWindows([1, 2, 1], [900, 40, 2000], causal=True, device=dev)
    q, k, v, _, _, _ = _inputs([1, 2, 1], [900, 40, 2000], 8, 2, 64, BF16, seed=23)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    with torch.no_grad():
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            packed_attention(q, k, v, win)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = packed_attention(q, k, v, win)
        for i in range(3):
            q.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, packed_attention(q, k, v, win))


@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_past_32_bits(dev, rows):
    """A cache of more than 2^31 elements; the last window's keys lie behind them."""
    H, d, kl = 16, 128, [1_050_000, 3000]
    g = torch.Generator(device=dev).manual_seed(12)
    k, v = (torch.empty(sum(kl), H, d, dtype=BF16, device=dev).normal_(generator=g) for _ in "kv")
    assert k.numel() > 2 ** 31
    q = torch.randn(rows, H, d, device=dev, generator=g).to(BF16)
    win = PackedWindows([0, rows], kl, causal=True, device=dev)
    with torch.no_grad():
        out = packed_attention(q, k, v, win)
    args = [t.cpu() for t in (q, k[kl[0]:], v[kl[0]:])]
    ref, bound = OP.bounds(*args, torch.zeros(rows, H, d), [rows], [3000], HALF[BF16], True)
    _check([out], ref, bound, "long cache")


def test_no_rows_and_no_windows(dev):
    for ql, kl in (([], []), ([0], [5]), ([3], [0])):
        win = PackedWindows(ql, kl, device=dev)
        q = torch.randn(sum(ql), 2, 16, device=dev, requires_grad=True)
        k, v = (torch.randn(sum(kl), 2, 16, device=dev, requires_grad=True) for _ in "kv")
        out = packed_attention(q, k, v, win)
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert out.shape == q.shape and not out.any() and not any(t.any() for t in grads)


def test_table_gradient_where_nothing_is_attended(dev):
    win = PackedWindows([3, 0], [0, 4], device=dev)
    q = torch.randn(3, 2, 16, device=dev)
    k = torch.randn(4, 2, 16, device=dev)
    t = torch.randn(5, 2, device=dev, requires_grad=True)
    b = win.pack_buckets(torch.empty(0, dtype=torch.uint8, device=dev))
    out = packed_attention(q, k, k, win, bias_table=t, buckets=b)
    assert not torch.autograd.grad(out.sum(), t)[0].any()


def test_second_derivatives_are_refused(dev):
    win = PackedWindows([20], device=dev)
    q, k, v = (torch.randn(20, 2, 16, device=dev, requires_grad=True) for _ in range(3))
    g, = torch.autograd.grad(packed_attention(q, k, v, win).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets", [0, 13])
def test_the_cpp_node_and_the_python_class_give_the_same_bits(dev, dtype, buckets, monkeypatch):
    assert _lib.autograd_ext() is not None
    ql = [70, 33, 1]
    q, k, v, go, table, ids = _inputs(ql, ql, 4, 2, 24, dtype, buckets, seed=30)
    win = PackedWindows(ql, causal=True, device=dev)
    a = _run(dev, q, k, v, go, table, ids, win)
    monkeypatch.setattr(_lib, "node_ext", lambda: None)
    b = _run(dev, q, k, v, go, table, ids, win)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    g, = torch.autograd.grad(
        packed_attention(x := q.to(dev).requires_grad_(), k.to(dev), v.to(dev), win).sum(), x,
        create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_gpu(dev):
    win = PackedWindows([5, 3], device=dev)
    q = torch.zeros(8, 4, 16, device=dev)
    k = torch.zeros(8, 2, 16, device=dev)
    b = win.pack_buckets(torch.zeros(34, dtype=torch.uint8, device=dev))
    t = torch.zeros(3, 4, device=dev)
    other = PackedWindows([5, 3], device=dev)
    bad = [((q[:7], k, k), {}, ValueError), ((q, k[:7], k[:7]), {}, ValueError),
           ((q, k, k[:, :1]), {}, ValueError), ((q, k.bfloat16(), k.bfloat16()), {}, TypeError),
           ((q.half(), k.half(), k.half()), {}, TypeError), ((q[:, :3], k, k), {}, ValueError),
           ((q[..., :12], k[..., :12], k[..., :12]), {}, ValueError),
           ((q, k.cpu(), k.cpu()), {}, ValueError), ((q, k, k), dict(scale=0.0), ValueError),
           ((q, k, k), dict(scale=math.inf), ValueError),
           ((q, k, k), dict(bias_table=t), ValueError), ((q, k, k), dict(buckets=b), ValueError),
           ((q, k, k), dict(bias_table=t.bfloat16(), buckets=b), ValueError),
           ((q, k, k), dict(bias_table=t[:, :2], buckets=b), ValueError),
           ((q, k, k), dict(bias_table=torch.zeros(256, 4, device=dev), buckets=b), ValueError),
           ((q, k, k), dict(bias_table=t[:0], buckets=b), ValueError)]
    for args, more, err in bad:
        with pytest.raises(err):
            packed_attention(*args, win, **more)
    with pytest.raises(ValueError, match="pack_buckets"):
        packed_attention(q, k, k, other, bias_table=t, buckets=b)
    for ids, err in ((torch.zeros(33, dtype=torch.uint8, device=dev), ValueError),
                     (torch.zeros(34, device=dev), TypeError),
                     (torch.zeros(34, dtype=torch.uint8), ValueError)):
        with pytest.raises(err):
            win.pack_buckets(ids)


def test_a_plan_made_and_dropped_on_another_stream(dev):
    """The plan's memory outlives the work that another stream still has to do."""
    ql = [300] * 20
    q, k, v, go, _, _ = _inputs(ql, ql, 4, 4, 32, BF16, seed=31)
    want = _run(dev, q, k, v, go, None, None, PackedWindows(ql, device=dev))
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    for _ in range(5):
        win = PackedWindows(ql, device=dev)
        n = win.mem.numel()
        with torch.cuda.stream(side), torch.no_grad():
            for _ in range(10):
                out = packed_attention(q, k, v, win)
        del win
        junk = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for _ in range(4)]
        side.synchronize()
        assert torch.equal(out, want[0])
        del junk


def test_ids_laid_out_and_dropped_on_another_stream(dev):
    """As above for the pairs' ids, whose memory is the side stream's."""
    ql = [600] * 4
    q, k, v, go, table, ids = _inputs(ql, ql, 4, 4, 16, BF16, 9, seed=32)
    win = PackedWindows(ql, device=dev)
    q, k, v, table, ids = (t.to(dev) for t in (q, k, v, table, ids))
    with torch.no_grad():
        want = packed_attention(q, k, v, win, bias_table=table, buckets=win.pack_buckets(ids))
        side = torch.cuda.Stream(dev)
        for _ in range(5):
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                b = win.pack_buckets(ids)
            torch.cuda.current_stream(dev).wait_stream(side)
            for _ in range(10):
                out = packed_attention(q, k, v, win, bias_table=table, buckets=b)
            n = b.by_query.numel()
            del b
            with torch.cuda.stream(side):
                junk = [torch.zeros(n, dtype=torch.uint8, device=dev) for _ in range(4)]
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            del junk


def test_two_graphs_and_eager_calls_of_one_plan(dev):
    """Two captured training steps of one plan, replayed in turn and side by side
    on two streams, with eager steps in between."""
    ql = [130, 7, 64]
    win = PackedWindows(ql, device=dev)
    sets = [[t.to(dev) for t in _inputs(ql, ql, 4, 2, 16, BF16, 12, seed=s)] for s in (40, 41)]
    b = win.pack_buckets(sets[0][5])

    def step(q, k, v, go, table, _):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
        out = packed_attention(*leaves[:3], win, bias_table=leaves[3], buckets=b)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, static = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            static.append(step(*s))
    side = torch.cuda.Stream(dev)
    for i in range(4):
        for x in (*static[0], *static[1]):
            x.zero_()
        side.wait_stream(torch.cuda.current_stream(dev))
        graphs[0].replay()
        with torch.cuda.stream(side) if i % 2 else torch.cuda.stream(torch.cuda.current_stream(dev)):
            graphs[1].replay()
        eager = step(*sets[i % 2])
        torch.cuda.synchronize()
        for a, w in ((static[0], want[0]), (static[1], want[1]), (eager, want[i % 2])):
            assert all(torch.equal(x, y) for x, y in zip(a, w))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_q,n_k", [(7, 300), (7, 2000), (200, 200)])
def test_rows_of_large_finite_table_entries(dev, dtype, n_q, n_k):
    """Masks of finite values: a row of nothing else weighs its greatest alike (scores of
    32 bits vanish beside them), any other row does not see them, in whichever order
    they come; and so do the gradients."""
    H, d = (4, 16) if n_q == 200 else (2, 16)
    far = [torch.finfo(dtype).min, -1e9, 1e9]
    q, k, v, go, table, _ = _inputs([n_q], [n_k], H, H, d, dtype, 6, seed=n_q, cut=0.0)
    for i, x in enumerate(far):
        table[i] = x
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(3, 6, (n_q, n_k), generator=g)  # of ordinary entries
    half_way = n_k // 2 + 3
    ids[0] = 0
    ids[1, :half_way] = 0
    ids[2] = 1
    ids[3, :half_way] = 1
    ids[4, :half_way], ids[4, half_way:] = 0, 1
    ids[5, half_way:] = 2
    ids[6, :70] = 1
    ids[6, 70:] = 255
    win = PackedWindows([n_q], [n_k], device=dev)
    got = _run(dev, q, k, v, go, table, ids.flatten(), win)

    u, half = 2.0 ** -24, HALF[dtype] if dtype == BF16 else 0.0
    Q, K, V, G = (t.double().transpose(0, 1) for t in (q, k, v, go))
    bias = table.double()[ids.clamp(max=5)].permute(2, 0, 1)
    s = Q @ K.transpose(1, 2) / math.sqrt(d)
    x = torch.where(bias.abs() > 1e8, bias, s + bias)
    x = x.masked_fill(ids == 255, -math.inf)
    p = torch.softmax(x, -1)
    small = torch.where(bias.abs() > 1e8, torch.zeros_like(bias), bias.abs())
    mag = Q.abs() @ K.abs().transpose(1, 2) / math.sqrt(d) + small
    # as oracle.packed.bounds, and 2^-15 of the weights: an ordinary row's base may be up to
    # 256 away from its products' start
    e_s = (((d + 4) * u * torch.where(p > 0, mag, 0.0)).amax(-1, keepdim=True)
           + (2.0 ** -15 if dtype == BF16 else 0.0))
    e_p = 2 * e_s + (n_k + 12) * u
    o = p @ V
    err_o = (e_p + half + n_k * u) * (p @ V.abs())
    dp = G @ V.transpose(1, 2)
    D = (G * o).sum(-1, keepdim=True)
    err_D = (G.abs() * err_o).sum(-1, keepdim=True) + d * u * (G * o).abs().sum(-1, keepdim=True)
    ds = p * (dp - D)
    err = p * (err_D + (d + 2) * u * (G.abs() @ V.abs().transpose(1, 2))) + (e_p + 4 * u) * ds.abs()
    r = err + half * (ds.abs() + err)
    sc, n = 1 / math.sqrt(d), max(n_q, n_k)
    ref = [o, sc * ds @ K, sc * ds.transpose(1, 2) @ Q, p.transpose(1, 2) @ G]
    bound = [err_o, sc * (r + (n + 2) * u * ds.abs()) @ K.abs(),
             sc * (r + (n + 2) * u * ds.abs()).transpose(1, 2) @ Q.abs(),
             ((e_p + half + n * u) * p).transpose(1, 2) @ G.abs()]
    one = torch.nn.functional.one_hot(ids, 256)[..., :6].double()
    ref = [t.transpose(0, 1) for t in ref] + [torch.einsum("hij,ijb->bh", ds, one)]
    bound = [t.transpose(0, 1) for t in bound]
    bound.append(torch.einsum("hij,ijb->bh", err + 4096 * u * ds.abs(), one))
    _check(got, ref, [b + HALF[dtype] * (t.abs() + b) for t, b in zip(ref, bound)], "far")
    assert (p[:, [0, 2]] - 1 / n_k).abs().max() < 1e-12
