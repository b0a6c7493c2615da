"""Packed attention and the linear epilogue on long windows and behind offsets of more
than 2^31 elements, forward and backward."""
import pytest
import torch

from neutrongt_amd import PackedWindows, linear_epilogue, packed_attention
from oracle import packed as OP
from tests.test_gpu_linear_epilogue import _ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
NAMES = ("out", "dq", "dk", "dv", "dtable")


def _check(got, ref, bound):
    for name, x, r, b in zip(NAMES, got, ref, bound):
        x = x.double().cpu()
        assert x.shape == r.shape and torch.isfinite(x).all(), name
        over = ((x - r).abs() - b).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ql,kl,H,hkv,d,buckets,causal", [
    ([2600, 900], [2600, 900], 2, 1, 16, 0, False), ([2500, 70], [2500, 70], 4, 2, 64, 0, True),
    ([2100], [2300], 2, 2, 128, 0, True), ([2600], [2600], 2, 2, 24, 40, False),
    ([30, 1900], [2900, 1900], 4, 4, 8, 200, True), ([3000], [20], 2, 2, 32, 0, False)])
def test_long_windows(dev, dtype, ql, kl, H, hkv, d, buckets, causal):
    print(f"case {ql} {kl} H={H}/{hkv} d={d} {dtype} {buckets}", flush=True)
    g = torch.Generator().manual_seed(d + buckets)
    q, go = (torch.randn(sum(ql), H, d, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(sum(kl), hkv, d, generator=g).to(dtype) for _ in range(2))
    win = PackedWindows(ql, kl, causal=causal, device=dev)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    table = ids = None
    more = {}
    if buckets:
        table = torch.randn(buckets, H, generator=g).to(dtype)
        ids = torch.randint(0, buckets, (sum(a * b for a, b in zip(ql, kl)),), generator=g)
        ids[torch.rand(ids.numel(), generator=g) < 0.05] = 255
        leaves.append(table.to(dev).requires_grad_())
        more = dict(bias_table=leaves[3], buckets=win.pack_buckets(ids.to(dev)))
    out = packed_attention(*leaves[:3], win, **more)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]
    _check(got, *OP.bounds(q, k, v, go, ql, kl, HALF[dtype], causal, None, table, ids))


@pytest.mark.parametrize("side", ["queries", "keys"])
def test_rows_behind_2_to_the_31(dev, side):
    """The second window's rows lie behind more than 2^31 elements of the first, which
    has nothing on the other side: zero rows, zero gradients."""
    H, d, far, n = 16, 128, 1_050_000, 40
    ql, kl = ([far, n], [0, n]) if side == "queries" else ([0, n], [far, n])
    assert far * H * d > 2 ** 31
    g = torch.Generator().manual_seed(4)
    small = [torch.randn(n, H, d, generator=g).to(BF16) for _ in range(4)]
    long = ("q", "go") if side == "queries" else ("k", "v")
    full = {}
    for name, t in zip(("q", "k", "v", "go"), small):
        x = torch.zeros((far if name in long else 0) + n, H, d, dtype=BF16, device=dev)
        x[-n:] = t.to(dev)
        full[name] = x
    leaves = [full[c].requires_grad_() for c in "qkv"]
    out = packed_attention(*leaves, PackedWindows(ql, kl, device=dev))
    got = [out.detach(), *torch.autograd.grad(out, leaves, full["go"])]
    for t in got:
        assert not t[:-n].any()
    q, k, v, go = small
    _check([t[-n:] for t in got], *OP.bounds(q, k, v, go, [n], [n], HALF[BF16]))


def test_bucket_ids_behind_2_to_the_31(dev):
    """The second window's ids lie behind more than 2^31 of the first's, whose output
    gradient is zero: it adds nothing to the table's gradient."""
    H, d, far, n = 2, 8, 46_400, 60
    lengths = [far, n]
    assert far * far > 2 ** 31
    g = torch.Generator().manual_seed(5)
    q, k, v, go = (torch.randn(far + n, H, d, generator=g).to(BF16) for _ in range(4))
    go[:far] = 0
    table = torch.randn(7, H, generator=g).to(BF16)
    ids = torch.zeros(far * far + n * n, dtype=torch.uint8, device=dev)
    last = torch.randint(0, 9, (n * n,), generator=g).to(torch.uint8)  # 7, 8: not in the table
    ids[-n * n:] = last.to(dev)
    win = PackedWindows(lengths, device=dev)
    packed = win.pack_buckets(ids)
    del ids
    rows = packed.by_query[-n * 64:].view(n, 64)[:, :n].cpu()
    assert torch.equal(rows.flatten(), last)
    assert torch.equal(packed.by_key[-n * 64:].view(n, 64)[:, :n].cpu(), rows.t())
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table)]
    out = packed_attention(*leaves[:3], win, bias_table=leaves[3], buckets=packed)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]
    assert all(torch.isfinite(t).all() for t in got)
    ref, bound = OP.bounds(q[far:], k[far:], v[far:], go[far:], [n], [n], HALF[BF16], False, None,
                           table, last)
    _check([t[far:] for t in got[:4]] + got[4:], ref, bound)


@pytest.mark.parametrize("n_out,n_in", [(24, 1032), (1032, 24)])
def test_linear_rows_behind_2_to_the_31(dev, n_out, n_in):
    """Rows of x or of y behind 2^31 elements; only the last have an output gradient."""
    far, n = 2_100_000, 50
    assert far * max(n_out, n_in) > 2 ** 31
    g = torch.Generator().manual_seed(6)
    xs, gy = torch.randn(n, n_in, generator=g).to(BF16), torch.randn(n, n_out, generator=g).to(BF16)
    w = (torch.randn(n_out, n_in, generator=g) / n_in ** 0.5).to(BF16)
    b = torch.randn(n_out, generator=g).to(BF16)
    x = torch.zeros(far + n, n_in, dtype=BF16, device=dev)
    x[far:] = xs.to(dev)
    gfull = torch.zeros(far + n, n_out, dtype=BF16, device=dev)
    gfull[far:] = gy.to(dev)
    leaves = [x.requires_grad_(), w.to(dev).requires_grad_(), b.to(dev).requires_grad_()]
    y = linear_epilogue(*leaves, activation="relu")
    dx, dw, db = torch.autograd.grad(y, leaves, gfull)
    first = torch.relu(b.double()).to(BF16)
    assert torch.equal(y[0].cpu(), first) and torch.equal(y[far - 1].cpu(), first)
    assert not dx[:far].any()
    ref = _ref(xs, w, b, None, gy, "relu")
    for name, t, (r, bound) in zip(("y", "dx", "dw", "db"), (y[far:], dx[far:], dw, db), ref):
        over = ((t.detach().double().cpu() - r).abs() - bound).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"
