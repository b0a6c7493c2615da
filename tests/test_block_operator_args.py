"""The C entries of the norm and rotation, the gated linear layer and the clipping refuse
bad arguments before anything is launched, and the formulas of the GPU tests' float64
references hold against differences (no GPU needed)."""
import ctypes as C
import math

import pytest
import torch

from neutrongt_amd import Rotary, _lib, clip_gradients, gated_linear, norm_rotary
from oracle import rotary as OR
from tests.test_gpu_gated_linear import _inputs, _ref

P = 1 << 20  # an address that nothing reads


def _heads(**kw):
    r = _lib.HeadRowsC(x=P, y=P, dy=P, x_row=64, x_head=16, dy_row=64, dy_head=16, n_heads=4)
    for n, v in kw.items():
        setattr(r, n, v)
    return r


def _rot(**kw):
    r = _lib.RotationC(P, P, 4, 16, 0, 1.0)
    for n, v in kw.items():
        setattr(r, n, v)
    return r


def test_norm_rotary_refusals_touch_no_gpu():
    lib = _lib.load()

    def fwd(dt=0, q=_heads(), k=None, n=4, d=16, rot=_rot(), eps=1e-6):
        ref = lambda s: C.byref(s) if s is not None else None
        return lib.ngt_norm_rotary_fwd(dt, ref(q), ref(k), n, d, ref(rot), eps, None)

    for bad, code in ((dict(dt=2), 1), (dict(n=-1), 1), (dict(n=(1 << 30) + 1), 1), (dict(d=15), 2),
                      (dict(d=0), 2), (dict(d=258), 2), (dict(q=None), 1), (dict(eps=-1.0), 1),
                      (dict(eps=math.nan), 1), (dict(rot=_rot(dim=-2)), 1), (dict(rot=_rot(dim=3)), 1),
                      (dict(rot=_rot(dim=18)), 1), (dict(rot=_rot(position_bytes=2)), 1),
                      (dict(rot=_rot(positions=None)), 1), (dict(rot=_rot(turns=None)), 1),
                      (dict(q=_heads(n_heads=0)), 1), (dict(k=_heads(n_heads=0)), 1),
                      (dict(q=_heads(x=None)), 1), (dict(q=_heads(y=None)), 1),
                      (dict(k=_heads(x=None)), 1), (dict(q=_heads(x_row=-1)), 1),
                      (dict(q=_heads(gain=P, gain_dtype=5)), 1)):
        assert fwd(**bad) == code, bad
        assert b"ngt_norm_rotary_fwd" in lib.ngt_last_error()
    assert fwd(n=0, q=_heads(x=None, y=None), rot=_rot(positions=None)) == 0

    def bwd(q=_heads(), ws=P, nb=1 << 20):
        return lib.ngt_norm_rotary_bwd(0, C.byref(q), None, 4, 16, C.byref(_rot()), 1e-6, ws, nb, None)

    nb = C.c_size_t()
    assert lib.ngt_norm_rotary_bwd_workspace_bytes(4, 16, C.byref(nb)) == 0 and nb.value > 0
    gain = dict(gain=P, dgain=P)
    for bad, code in ((dict(q=_heads(dy=None)), 1), (dict(q=_heads(dgain=P)), 1),
                      (dict(q=_heads(x=None, gain=P)), 1),
                      (dict(q=_heads(**gain), ws=None), 4), (dict(q=_heads(**gain), nb=nb.value - 1), 4),
                      (dict(q=_heads(**gain), ws=P + 8), 4)):
        assert bwd(**bad) == code, bad
        assert b"ngt_norm_rotary_bwd" in lib.ngt_last_error()
    for args in ((-1, 16), (4, 0), (4, 258), ((1 << 30) + 1, 16)):
        assert lib.ngt_norm_rotary_bwd_workspace_bytes(*args, C.byref(nb)) == 1


def test_gated_refusals_touch_no_gpu():
    lib = _lib.load()

    def fwd(x=P, xs=8, wg=P, wu=P, rows=4, n_out=6, n_in=8, act=3, y=P, keep=None, ws=None, nb=0):
        return lib.ngt_gated_fwd(x, xs, wg, wu, None, None, rows, n_out, n_in, act, y, keep, ws, nb,
                                 None)

    for bad, code in ((dict(rows=-1), 1), (dict(n_out=0), 1), (dict(n_in=0), 1), (dict(act=4), 1),
                      (dict(act=-1), 1), (dict(x=None), 1), (dict(wg=None), 1), (dict(wu=None), 1),
                      (dict(y=None), 1), (dict(xs=7), 1), (dict(keep=P + 8), 1),
                      (dict(rows=(1 << 30) + 1), 2), (dict(rows=1 << 30, n_out=1 << 12), 2),
                      (dict(n_out=(1 << 29) + 1), 2), (dict(n_out=1 << 20), 2),
                      (dict(xs=1 << 21, n_in=1 << 21), 2)):
        assert fwd(**bad) == code, bad
        assert b"ngt_gated_fwd" in lib.ngt_last_error()
    assert fwd(rows=0, x=None, y=None) == 0
    nb = C.c_size_t()
    for size in ((4, 6, 8), (0, 64, 8192), (100000, 64, 8192)):
        assert lib.ngt_gated_fwd_workspace_bytes(*size, C.byref(nb)) == 0 and nb.value == 0
    assert lib.ngt_gated_fwd_workspace_bytes(4, 0, 8, C.byref(nb)) == 1
    for rows in (1, 100):
        assert lib.ngt_gated_fwd_workspace_bytes(rows, 64, 8192, C.byref(nb)) == 0 and nb.value > 0
        long = dict(xs=8192, rows=rows, n_out=64, n_in=8192)
        for bad in (dict(nb=nb.value), dict(ws=P, nb=nb.value - 1), dict(ws=P + 8, nb=nb.value)):
            assert fwd(**long, **bad) == 4, bad
    assert lib.ngt_gated_keep_bytes(4, 6, C.byref(nb)) == 0 and nb.value >= 4 * 6 * 2 * 2
    assert lib.ngt_gated_keep_bytes(-1, 6, C.byref(nb)) == 1
    assert lib.ngt_gated_bwd_workspace_bytes(4, 6, 8, C.byref(nb)) == 0

    def bwd(dy=P, keep=P, x=P, wg=P, wu=P, ws=P, n=nb.value, grads=True, **kw):
        g = _lib.GatedGradsC(P, P, P, P, P, 0, 1, 0, 1)
        for name, v in kw.items():
            setattr(g, name, v)
        return lib.ngt_gated_bwd(dy, keep, x, wg, wu, 4, 6, 8, C.byref(g) if grads else None, ws, n,
                                 None)

    for bad, code in ((dict(dy=None), 1), (dict(keep=None), 1), (dict(x=None), 1), (dict(wg=None), 1),
                      (dict(wu=None), 1), (dict(grads=False), 1), (dict(dw_gate_dtype=4), 1),
                      (dict(db_up_dtype=-1), 1), (dict(dw_up=P + 8), 1), (dict(x=P + 2), 1),
                      (dict(wu=P + 8), 1), (dict(dy=P + 2), 1), (dict(dx=P + 4), 1), (dict(ws=None), 4),
                      (dict(n=nb.value - 1), 4), (dict(ws=P + 8), 4)):
        assert bwd(**bad) == code, bad
        assert b"ngt_gated_bwd" in lib.ngt_last_error()


def test_clip_refusals_touch_no_gpu():
    lib = _lib.load()
    nb = C.c_size_t()

    def run(max_norm=1.0, norm=P, ws=P, size=1 << 20, n=1, **kw):
        t = (_lib.GradientC * 1)(_lib.GradientC(P, None, 8, 0, 0))
        for name, v in kw.items():
            setattr(t[0], name, v)
        return lib.ngt_clip_gradients(t, n, max_norm, norm, ws, size, None)

    for bad, code in ((dict(max_norm=math.nan), 1), (dict(norm=None), 1), (dict(ws=None), 4),
                      (dict(ws=P + 8), 4), (dict(size=23), 4), (dict(n=-1), 1), (dict(x=None), 1),
                      (dict(dtype=3), 1), (dict(out=P * 2, out_dtype=7), 1), (dict(x=P + 2), 1),
                      (dict(out=P + 1, out_dtype=1), 1), (dict(out=P, out_dtype=1), 1)):
        assert run(**bad) == code, bad
        assert b"ngt_clip_gradients" in lib.ngt_last_error()
    t = (_lib.GradientC * 1)(_lib.GradientC(P, None, -1, 0, 0))
    assert lib.ngt_clip_workspace_bytes(t, 1, C.byref(nb)) == 1


def test_python_entries_take_no_cpu_tensors():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError):
        gated_linear(x, w, w)
    with pytest.raises(ValueError):
        norm_rotary(torch.zeros(4, 2, 8))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError):
        clip_gradients([p], 1.0)
    assert torch.equal(p.grad, torch.ones(3))


@pytest.mark.parametrize("kw", [dict(dim=3), dict(dim=-2), dict(layout="pairs"),
                                dict(scaling="ntk"), dict(factor=0.0), dict(base=-1.0),
                                dict(base=math.inf), dict(frequencies=[1.0]),
                                dict(frequencies=[1.0] * 7 + [math.nan]), dict(scaling="parts"),
                                dict(scaling="parts", trained_length=64, slow=2.0, fast=2.0),
                                dict(magnitude=math.inf), dict(device="cpu")])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        Rotary(**{"dim": 16, **kw})


def _differences(loss, tensors, grads, tol):
    for t, got in zip(tensors, grads):
        at = t.view(-1)
        for i in range(t.numel()):
            keep, h = at[i].item(), 1e-5
            at[i] = keep + h
            up = loss()
            at[i] = keep - h
            down = loss()
            at[i] = keep
            assert abs((up - down) / (2 * h) - got.reshape(-1)[i].item()) < tol


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_the_formulas_of_the_gated_gradients_against_differences(act):
    """Central differences of the reference's forward (step 1e-5: truncation 1e-10,
    rounding 1e-11)."""
    x, wg, wu, bg, bu, gy = (t.double() for t in _inputs(5, 4, 6, True, 2))

    def loss():
        return (_ref(x, wg, wu, bg, bu, gy, act)[0][0] * gy).sum().item()

    grads = [g for g, _ in _ref(x, wg, wu, bg, bu, gy, act)[1:]]
    _differences(loss, (x, wg, wu, bg, bu), grads, 1e-7)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_rotary_reference(layout):
    """Its gradients against differences; and what a rotation has to do: scores of turned
    queries and keys depend on the distance of their positions alone, and a full turn
    is none."""
    g = torch.Generator().manual_seed(0)
    x, gy = (torch.randn(3, 2, 10, generator=g, dtype=torch.float64) for _ in range(2))
    gain = 1 + 0.1 * torch.randn(10, generator=g, dtype=torch.float64)
    pos, f = torch.tensor([0, 5, -3]), torch.tensor([1.0, 0.3, 0.01], dtype=torch.float64)

    def loss():
        return (OR.forward(x, gain, pos, f, layout, 1.3) * gy).sum().item()

    ref = OR.bounds(x, gain, pos, f, layout, 1.3, 1e-6, gy, 0.0, 0.0)
    _differences(loss, (x, gain), (ref[1][0], ref[2][0]), 1e-7)
    q, k = x[:1, :1], x[1:2, 1:]
    score = lambda i, j: (OR.forward(q, None, torch.tensor([i]), f, layout)
                          * OR.forward(k, None, torch.tensor([j]), f, layout)).sum().item()
    assert abs(score(7, 3) - score(104, 100)) < 1e-12 and abs(score(7, 3) - score(7, 4)) > 1e-3
    turn = OR.forward(x, None, torch.tensor([4, 8, 12]), torch.full((3,), math.pi / 2,
                                                                    dtype=torch.float64), layout)
    assert torch.allclose(turn, x, rtol=0, atol=1e-12)
