"""The few-query form of packed attention: 16 bits of every weight in bf16, wide heads
and large groups with a bias, one split and many."""
import math

import pytest
import torch

from neutrongt_amd import PackedWindows, packed_attention
from oracle import packed as OP

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def _inputs(ql, kl, H, hkv, d, dtype, buckets, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(ql), H, d, generator=g).to(dtype)
    k, v = (torch.randn(sum(kl), hkv, d, generator=g).to(dtype) for _ in range(2))
    table = ids = None
    if buckets:
        table = torch.randn(buckets, H, generator=g).to(dtype)
        ids = torch.randint(0, buckets, (sum(a * b for a, b in zip(ql, kl)),), generator=g)
    return q, k, v, table, ids


@pytest.mark.parametrize("d", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("ql,kl", [([1, 1], [200, 700]), ([1], [4000]), ([4, 2], [900, 150])])
@pytest.mark.parametrize("buckets", [0, 9])
def test_bf16_weights_keep_16_bits(dev, d, ql, kl, buckets):
    """The bound of an unrounded weight (oracle.packed.bounds of fp32, whose result is
    off by err), 2^-16 of each weight (its two pieces), and the result's half step."""
    q, k, v, table, ids = _inputs(ql, kl, 8, 2, d, BF16, buckets, d)
    win = PackedWindows(ql, kl, causal=True, device=dev)
    more = {} if table is None else dict(bias_table=table.to(dev),
                                         buckets=win.pack_buckets(ids.to(dev)))
    out = packed_attention(q.to(dev), k.to(dev), v.to(dev), win, **more).double().cpu()
    ref, bound = OP.bounds(q, k, v, torch.zeros_like(q), ql, kl, 2.0 ** -24, True, None, table, ids)
    weighed = OP.attention(q.double(), k.double(), v.double().abs(), ql, kl, True, None,
                           table.double() if buckets else None, ids)
    err = bound[0] + 2.0 ** -16 * weighed
    err = err + HALF[BF16] * (ref[0].abs() + err)
    over = ((out - ref[0]).abs() - err).max().item()
    assert over <= 0, f"{over:.3e} over the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [72, 128])
@pytest.mark.parametrize("H,hkv", [(4, 4), (32, 1)])
@pytest.mark.parametrize("nk", [300, 4000])
def test_wide_heads_and_large_groups_with_a_bias(dev, dtype, d, H, hkv, nk):
    """Up to 66,560 bytes of tiles and a table of every head of the group in LDS (96 KB)."""
    print(f"case d={d} H={H}/{hkv} keys={nk} {dtype}", flush=True)
    ql, kl = [1, 0, 1], [nk, 7, 140]
    q, k, v, table, ids = _inputs(ql, kl, H, hkv, d, dtype, 255, d + H)
    win = PackedWindows(ql, kl, device=dev)
    g = torch.Generator().manual_seed(3)
    go = torch.randn(q.shape, generator=g).to(dtype)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table)]
    out = packed_attention(*leaves[:3], win, bias_table=leaves[3],
                           buckets=win.pack_buckets(ids.to(dev)))
    got = [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]
    ref, bound = OP.bounds(q, k, v, go, ql, kl, HALF[dtype], False, 1 / math.sqrt(d), table, ids)
    for name, x, r, b in zip(("out", "dq", "dk", "dv", "dtable"), got, ref, bound):
        over = ((x.double().cpu() - r).abs() - b).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"
