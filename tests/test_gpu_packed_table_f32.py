"""An fp32 bias table beside bf16 rows, as a training step under autocast has it: the
learned table goes in unrounded, and its gradient comes out in fp32."""
import ctypes as C

import pytest
import torch

from neutrongt_amd import PackedWindows, _lib, packed_attention
from neutrongt_amd.linear import WgradLinear, project
from oracle import packed as OP

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HB, U = 2.0 ** -8, 2.0 ** -24


def _inputs(ql, kl, H, hkv, d, buckets, seed):
    g = torch.Generator().manual_seed(seed)
    q, go = (torch.randn(sum(ql), H, d, generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(sum(kl), hkv, d, generator=g).to(BF16) for _ in range(2))
    table = torch.randn(buckets, H, generator=g)  # not values of bf16
    n = sum(a * b for a, b in zip(ql, kl))
    ids = torch.randint(0, buckets, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.05] = 255
    return q, k, v, go, table, ids


def _run(dev, q, k, v, go, table, ids, win):
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table)]
    out = packed_attention(*leaves[:3], win, bias_table=leaves[3],
                           buckets=win.pack_buckets(ids.to(dev)))
    return [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]


@pytest.mark.parametrize("lengths,H,hkv,d,buckets,causal", [
    (([70, 3, 30], [70, 3, 30]), 4, 4, 8, 7, False), (([65, 129], [65, 129]), 8, 8, 24, 64, True),
    (([50, 20], [130, 20]), 6, 2, 64, 65, True), (([100, 1], [100, 1]), 2, 2, 128, 255, False),
    (([1, 2, 1], [300, 140, 1]), 8, 2, 32, 31, False), (([1, 1], [4000, 130]), 8, 8, 64, 12, True),
    (([30], [25]), 4, 4, 32, 9, False), (([400, 100], [400, 130]), 64, 64, 16, 40, True)])
def test_against_float64(dev, lengths, H, hkv, d, buckets, causal):
    """The bounds of bf16 rows; the table's gradient rounded to fp32, not to bf16."""
    args = _inputs(*lengths, H, hkv, d, buckets, buckets)
    win = PackedWindows(*lengths, causal=causal, device=dev)
    got = _run(dev, *args, win)
    assert got[4].dtype == F32 and all(t.dtype == BF16 for t in got[:4])
    ref, bound = OP.bounds(*args[:4], *lengths, HB, causal, None, *args[4:])
    sums = (bound[4] - HB * ref[4].abs()) / (1 + HB)  # before the rounding of the result
    bound[4] = sums + U * (ref[4].abs() + sums)
    for name, x, r, b in zip(("out", "dq", "dk", "dv", "dtable"), got, ref, bound):
        x = x.double().cpu()
        assert x.shape == r.shape and torch.isfinite(x).all(), name
        over = ((x - r).abs() - b).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"


def test_a_table_of_bf16_values_gives_the_same_rows_in_either_type(dev):
    ql = [70, 33, 1]
    q, k, v, go, table, ids = _inputs(ql, ql, 4, 2, 24, 13, 5)
    win = PackedWindows(ql, causal=True, device=dev)
    a = _run(dev, q, k, v, go, table.to(BF16), ids, win)
    b = _run(dev, q, k, v, go, table.to(BF16).float(), ids, win)
    assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))
    assert torch.equal(a[4], b[4].to(BF16))


def test_the_cpp_node_and_the_python_class_give_the_same_bits(dev, monkeypatch):
    assert _lib.autograd_ext() is not None
    ql = [70, 33, 1]
    args = _inputs(ql, ql, 4, 2, 24, 13, 6)
    win = PackedWindows(ql, device=dev)
    a = _run(dev, *args, win)
    monkeypatch.setattr(_lib, "node_ext", lambda: None)
    b = _run(dev, *args, win)
    assert all(torch.equal(x, y) and x.dtype == y.dtype for x, y in zip(a, b))


def test_a_parameter_under_autocast(dev):
    """q, k and v of a joint projection in bf16, the table an fp32 parameter."""
    torch.manual_seed(0)
    lengths, H, d = [40, 25], 4, 16
    x = torch.randn(65, H * d, device=dev, requires_grad=True)
    lin = [WgradLinear(H * d, H * d).to(dev) for _ in range(3)]
    spatial_pos = torch.nn.Embedding(11, H).to(dev)
    win = PackedWindows(lengths, device=dev)
    ids = win.pack_buckets([torch.randint(0, 11, (n, n), device=dev) for n in lengths])
    with torch.autocast("cuda", dtype=BF16):
        q, k, v = (t.view(65, H, d) for t in project(x, *lin))
        assert q.dtype == BF16
        out = packed_attention(q, k, v, win, bias_table=spatial_pos.weight, buckets=ids)
    out.float().sum().backward()
    g = spatial_pos.weight.grad
    assert g.dtype == F32 and torch.isfinite(g).all() and g.abs().max() > 0


def test_refusals(dev):
    win = PackedWindows([5, 3], device=dev)
    ids = win.pack_buckets(torch.zeros(34, dtype=torch.uint8, device=dev))
    q = torch.zeros(8, 4, 16, device=dev, dtype=BF16)
    for table, rows in ((torch.zeros(3, 4, device=dev, dtype=BF16), q.float()),
                        (torch.zeros(3, 4, device=dev, dtype=torch.float64), q),
                        (torch.zeros(3, 4, device=dev, dtype=torch.float16), q),
                        (torch.zeros(3, 4), q)):
        with pytest.raises(ValueError, match="bias_table"):
            packed_attention(rows, rows, rows, win, bias_table=table, buckets=ids)


def test_the_flag_in_the_c_entries(dev):
    """fp32 rows take it as well (their table is fp32 anyway); other bits are refused."""
    lib, ql = _lib.load(), [9]
    win = PackedWindows(ql, device=dev)
    q, table = torch.randn(9, 2, 16, device=dev), torch.randn(3, 2, device=dev)
    b = win.pack_buckets(torch.randint(0, 3, (81,), device=dev))
    out = [torch.zeros_like(q) for _ in range(2)]
    call = lambda dtype, o: lib.ngt_packed_fwd(
        dtype, q.data_ptr(), q.data_ptr(), q.data_ptr(), 32, 32, 32, win.ptr(), 2, 2, 16, 0.25,
        table.data_ptr(), 3, b.by_query.data_ptr(), o.data_ptr(), None, None, None, 0,
        _lib.stream_ptr(dev))
    assert call(0, out[0]) == 0 and call(_lib.NGT_TABLE_F32, out[1]) == 0
    assert torch.equal(*out)
    nb = C.c_size_t()
    for bad in (0x200, 0x102, 2):
        assert call(bad, out[0]) == 1
        assert lib.ngt_packed_workspace_bytes(bad, win.ptr(), 2, 2, 16, 0, C.byref(nb), None) == 1
