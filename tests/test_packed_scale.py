"""The range of packed attention's scale: refused outside of it before anything is
launched, and right at its small end."""
import ctypes as C

import pytest
import torch

from neutrongt_amd import PackedWindows, _lib, packed_attention
from oracle import packed as OP
from tests.test_packed_args import _plan

P = 1 << 20  # an address that nothing reads
OUTSIDE = [0.0, -1.0, 1e-45, 1e-40, 2.0 ** -101, 2.0 ** 101, 3e38, float("inf"), float("nan")]


@pytest.mark.parametrize("scale", OUTSIDE)
@pytest.mark.parametrize("dtype", [0, 1])
def test_the_c_entries_refuse_it(scale, dtype):
    lib = _lib.load()
    st, _ = _plan([40], [300], 0)
    w = C.byref(st)
    for table in (None, P):
        nb = 3 if table else 0
        assert lib.ngt_packed_fwd(dtype, P, P, P, 32, 32, 32, w, 2, 2, 16, scale, table, nb, table,
                                  P, None, None, None, 0, None) == 1
        assert b"scale" in lib.ngt_last_error()
        assert lib.ngt_packed_bwd(dtype, P, P, P, 32, 32, 32, P, P, P, w, 2, 2, 16, scale, table,
                                  nb, table, table, P, P, P, None, None, 0, None) == 1
        assert b"scale" in lib.ngt_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", OUTSIDE + [1e-50, 1e50])
def test_python_refuses_it(dev, scale, monkeypatch):
    win = PackedWindows([5], device=dev)
    q = torch.zeros(5, 2, 16, device=dev)
    for _ in range(2):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, q, q, win, scale=scale)
        monkeypatch.setattr(_lib, "node_ext", lambda: None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scale", [2.0 ** -100, 1e-20, 1e-3, 3.0])
def test_small_scales(dev, dtype, nq, bias, scale):
    """Within the bounds of every scale.  dq and dk are as small as the scale, so that
    they are checked times 1 / scale."""
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
    g = torch.Generator().manual_seed(2)
    nk = 300
    q, go = (torch.randn(nq, 2, 16, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(nk, 2, 16, generator=g).to(dtype) for _ in range(2))
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    win = PackedWindows([nq], [nk], device=dev)
    table = ids = None
    more = {}
    if bias:
        table = torch.randn(5, 2, generator=g).to(dtype)
        ids = torch.randint(0, 5, (nq * nk,), generator=g)
        leaves.append(table.to(dev).requires_grad_())
        more = dict(bias_table=leaves[3], buckets=win.pack_buckets(ids.to(dev)))
    out = packed_attention(*leaves[:3], win, scale=scale, **more)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go.to(dev))]
    ref, bound = OP.bounds(q, k, v, go, [nq], [nk], half, False, scale, table, ids)
    for i, (x, r, b) in enumerate(zip(got, ref, bound)):
        by = 1 / scale if i in (1, 2) else 1.0
        assert ((x.double().cpu() - r).abs() * by <= b * by).all(), i
