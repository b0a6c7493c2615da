"""ngt_linear_fwd / ngt_linear_bwd refuse bad arguments before anything is
launched (no GPU needed)."""
import ctypes as C

import pytest

from neutrongt_amd import _lib
from tests.test_gpu_linear_epilogue import _inputs, _ref

P = 1 << 20  # an address that nothing reads


def test_refusals_touch_no_gpu():
    lib = _lib.load()

    def fwd(x=P, xs=8, w=P, rows=4, n_out=6, n_in=8, act=0, y=P):
        return lib.ngt_linear_fwd(x, xs, w, None, None, rows, n_out, n_in, act, y, None, None)

    for bad, code in ((dict(rows=-1), 1), (dict(n_out=0), 1), (dict(n_in=0), 1), (dict(act=3), 1),
                      (dict(act=-1), 1), (dict(x=None), 1), (dict(w=None), 1), (dict(y=None), 1),
                      (dict(xs=7), 1), (dict(rows=(1 << 30) + 1), 2),
                      (dict(rows=1 << 30, n_out=1 << 12), 2),
                      (dict(n_out=1 << 20, n_in=1 << 20, xs=1 << 20), 2)):
        assert fwd(**bad) == code, bad
        assert b"ngt_linear_fwd" in lib.ngt_last_error()
    assert fwd(rows=0, x=None, y=None) == 0

    def bwd(dy=P, z=P, w=P, act=2, dz=P, dx=P, ws=P, n=96):
        return lib.ngt_linear_bwd(dy, z, w, 4, 6, 8, act, dz, dx, ws, n, None)

    nb = C.c_size_t()
    assert lib.ngt_linear_bwd_workspace_bytes(4, 6, 8, C.byref(nb)) == 0 and nb.value == 96
    for bad, code in ((dict(dy=None), 1), (dict(z=None), 1), (dict(dz=None), 1), (dict(w=None), 1),
                      (dict(act=5), 1), (dict(dy=P + 2), 1), (dict(z=P + 2), 1),
                      (dict(dz=P + 8), 1), (dict(ws=None), 4), (dict(n=95), 4), (dict(ws=P + 8), 4)):
        assert bwd(**bad) == code, bad
        assert b"ngt_linear_bwd" in lib.ngt_last_error()


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
def test_the_formulas_of_the_gradients_against_differences(act):
    """The float64 reference of the GPU tests: every gradient against central
    differences of its forward (step 1e-5: truncation 1e-10, rounding 1e-11)."""
    x, w, b, r, gy = (t.double() for t in _inputs(5, 4, 6, True, True, 2))

    def loss():
        return (_ref(x, w, b, r, gy, act)[0][0] * gy).sum().item()

    for t, (got, _) in zip((x, w, b), _ref(x, w, b, r, gy, act)[1:]):
        for i in range(t.numel()):
            at, h = t.view(-1), 1e-5
            keep = at[i].item()
            at[i] = keep + h
            up = loss()
            at[i] = keep - h
            down = loss()
            at[i] = keep
            assert abs((up - down) / (2 * h) - got.reshape(-1)[i].item()) < 1e-7
