"""Packed attention on NaN and infinities: every result that depends on one by the
formula shows it, no other result does."""
import math

import pytest
import torch

from neutrongt_amd import PackedWindows, packed_attention
from oracle import packed as OP

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _inputs(nq, nk, H, hkv, d, dtype, bias):
    g = torch.Generator().manual_seed(1)
    q, go = (torch.randn(nq, H, d, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(nk, hkv, d, generator=g).to(dtype) for _ in range(2))
    table = torch.randn(5, H, generator=g).to(dtype) if bias else None
    ids = torch.randint(0, 5, (nq * nk,), generator=g) if bias else None
    return q, k, v, go, table, ids


def _run(dev, q, k, v, go, table, ids, win):
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    more = {}
    if table is not None:
        leaves.append(table.to(dev).requires_grad_())
        more = dict(bias_table=leaves[3], buckets=win.pack_buckets(ids.to(dev)))
    out = packed_attention(*leaves[:3], win, **more)
    return [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]


# one query with one split and with many, a group's, block forms of one and more sets
SHAPES = [(1, 200, 2, 2, 16), (1, 4000, 2, 1, 16), (1, 4000, 2, 2, 128), (3, 4000, 8, 2, 64),
          (20, 30, 2, 2, 32), (40, 300, 2, 2, 16), (300, 300, 2, 2, 64), (700, 700, 2, 2, 16),
          (60, 60, 4, 2, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_nan_reaches_what_depends_on_it(dev, dtype, bias, shape):
    """All pairs are seen, so the float64 formula's NaN are the ones there must be: of a
    NaN in a key, the rows' weights of all keys and with them v's gradient."""
    nq, nk = shape[:2]
    win = PackedWindows([nq], [nk], device=dev)
    for at in range(4):  # q, k, v, the output's gradient
        q, k, v, go, table, ids = _inputs(*shape, dtype, bias)
        t = (q, k, v, go)[at]
        t[t.shape[0] // 2, -1, 3] = math.nan
        got = _run(dev, q, k, v, go, table, ids, win)
        want = OP.fwd_bwd(q, k, v, go, [nq], [nk], False, None, table, ids)
        for name, a, b in zip(("out", "dq", "dk", "dv", "dtable"), got, want):
            assert torch.equal(a.isnan().cpu(), b.isnan()), f"NaN in {'qkvg'[at]}: {name}"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 4000, 2, 1, 16), (40, 300, 2, 2, 16), (300, 300, 2, 2, 128)])
def test_a_nan_in_a_row_of_large_table_entries(dev, dtype, shape):
    """The same where the rows keep their base and the logarithm of their sum apart."""
    nq, nk = shape[:2]
    win = PackedWindows([nq], [nk], device=dev)
    q, k, v, go, table, ids = _inputs(*shape, dtype, True)
    table[0] = -1e9
    ids.fill_(0)
    k[nk // 2, -1, 3] = math.nan
    got = _run(dev, q, k, v, go, table, ids, win)
    want = OP.fwd_bwd(q, k, v, go, [nq], [nk], False, None, table, ids)
    for name, a, b in zip(("out", "dq", "dk", "dv", "dtable"), got, want):
        assert torch.equal(a.isnan().cpu(), b.isnan()), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_an_infinite_value_is_not_lost(dev, dtype, shape):
    """Infinite v: every row weighs it, so the column is not finite (where operands are
    split into pieces it may come out as NaN); the other columns are as without it."""
    nq, nk, H, hkv, d = shape
    win = PackedWindows([nq], [nk], device=dev)
    q, k, v, _, _, _ = _inputs(*shape, dtype, False)
    run = lambda: packed_attention(q.to(dev), k.to(dev), v.to(dev), win)
    want = run()
    v[nk // 3, 0, 5] = math.inf
    got = run()
    heads = H // hkv
    assert not torch.isfinite(got[:, :heads, 5]).any()
    rest = torch.ones(H, d, dtype=torch.bool, device=dev)
    rest[:heads, 5] = False
    assert torch.equal(got[:, rest], want[:, rest])
