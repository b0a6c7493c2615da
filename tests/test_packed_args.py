"""Packed windows without a GPU: the host plan, and what is refused before
anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from neutrongt_amd import PackedWindows, _lib, packed_attention

BASE = 1 << 40  # stands for a device address


def _plan(ql, kl, causal):
    lib = _lib.load()
    a, b = np.array(ql, np.int32), np.array(kl, np.int32)
    nb, st = C.c_size_t(), _lib.PackedWindowsC()
    _lib.check(lib.ngt_packed_plan_bytes(len(a), a.ctypes.data, b.ctypes.data, C.byref(nb)))
    host = np.full(nb.value, 0x55, np.uint8)
    _lib.check(lib.ngt_packed_plan(len(a), a.ctypes.data, b.ctypes.data, causal, host.ctypes.data,
                                   nb.value, BASE, C.byref(st)))

    def at(p, n, t):
        return host[p - BASE:p - BASE + n * np.dtype(t).itemsize].view(t)

    return st, at


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("ql,kl", [([70, 3, 30], [70, 3, 30]), ([0, 5], [9, 0]), ([], []),
                                   ([1] * 40, [500] * 40), ([300, 1, 129], [20, 4000, 128])])
def test_plan(ql, kl, causal):
    st, at = _plan(ql, kl, causal)
    n = len(ql)
    up = lambda x: (x + 63) // 64 * 64
    want = {"q_start": ql, "k_start": kl, "p_start": [a * b for a, b in zip(ql, kl)],
            "b_start": [a * up(b) for a, b in zip(ql, kl)],
            "bt_start": [b * up(a) for a, b in zip(ql, kl)]}
    for f, lens in want.items():
        assert at(getattr(st, f), n + 1, np.int64).tolist() == [0] + np.cumsum(lens).tolist()
    assert (st.n_q, st.n_k, st.max_q, st.max_k) == (sum(ql), sum(kl), max(ql, default=0),
                                                    max(kl, default=0))
    for lens, other, items, counts, keys in ((ql, kl, st.items_q, st.n_items_q, False),
                                             (kl, ql, st.items_k, st.n_items_k, True)):
        for i, rows in enumerate((32, 64, 128)):
            got = at(items[i], 2 * counts[i], np.int32).reshape(-1, 2).tolist()
            assert sorted(got) == [[w, r] for w in range(n) for r in range(0, lens[w], rows)]

            def steps(w, r):
                seen = other[w]
                if causal:
                    seen = (ql[w] - max(0, r - (kl[w] - ql[w])) if keys
                            else min(min(r + rows, ql[w]) + kl[w] - ql[w], kl[w]))
                return (max(0, min(seen, other[w])) + 63) // 64

            cost = [steps(w, r) for w, r in got]
            assert cost == sorted(cost, reverse=True)


def test_plan_refusals():
    lib = _lib.load()
    one, neg, big = (np.array([x], np.int32) for x in (4, -1, (1 << 28) + 1))
    nb, st = C.c_size_t(), _lib.PackedWindowsC()
    assert lib.ngt_packed_plan_bytes(1, neg.ctypes.data, one.ctypes.data, C.byref(nb)) == 1
    assert lib.ngt_packed_plan_bytes(1, one.ctypes.data, big.ctypes.data, C.byref(nb)) == 2
    assert lib.ngt_packed_plan_bytes(1, None, one.ctypes.data, C.byref(nb)) == 1
    assert lib.ngt_packed_plan_bytes(-1, one.ctypes.data, one.ctypes.data, C.byref(nb)) == 1
    assert lib.ngt_packed_plan_bytes(1, one.ctypes.data, one.ctypes.data, C.byref(nb)) == 0
    host = np.zeros(nb.value, np.uint8)
    assert lib.ngt_packed_plan(1, one.ctypes.data, one.ctypes.data, 0, host.ctypes.data,
                               nb.value - 1, BASE, C.byref(st)) == 4
    assert lib.ngt_packed_plan(1, one.ctypes.data, one.ctypes.data, 0, host.ctypes.data, nb.value,
                               BASE, None) == 1


def test_call_refusals_touch_no_gpu():
    lib = _lib.load()
    st, _ = _plan([40], [300], 0)
    w = C.byref(st)
    p = 1 << 20  # a 16-byte aligned address that nothing reads

    def fwd(dtype=1, q=p, k=p, v=p, sq=32, sk=32, sv=32, win=w, H=2, hkv=2, d=16, scale=1.0,
            table=None, nb=0, ids=None, out=p, ws=None, n=0):
        return lib.ngt_packed_fwd(dtype, q, k, v, sq, sk, sv, win, H, hkv, d, scale, table, nb, ids,
                                  out, None, None, ws, n, None)

    for bad, code in ((dict(dtype=5), 1), (dict(win=None), 1), (dict(H=0), 1), (dict(hkv=0), 1),
                      (dict(H=3), 1), (dict(d=12), 2), (dict(d=136), 2), (dict(d=0), 2),
                      (dict(scale=0.0), 1), (dict(scale=float("nan")), 1),
                      (dict(scale=float("inf")), 1), (dict(q=None), 1), (dict(k=None), 1),
                      (dict(v=None), 1), (dict(out=None), 1), (dict(sq=31), 1), (dict(sk=36), 1),
                      (dict(q=p + 8), 1),
                      (dict(sk=1 << 22), 2), (dict(H=40000, hkv=40000, d=128), 2), (dict(table=p), 1), (dict(ids=p), 1),
                      (dict(table=p, ids=p, nb=0), 1), (dict(table=p, ids=p, nb=256), 1)):
        assert fwd(**bad) == code, bad
        assert b"ngt_packed_fwd" in lib.ngt_last_error()
    long, _ = _plan([4], [(1 << 23) + 1], 0)
    assert fwd(win=C.byref(long), table=p, ids=p, nb=3) == 2
    few, _ = _plan([1], [100000], 1)  # splits its keys: needs a workspace
    fb = C.c_size_t()
    assert lib.ngt_packed_workspace_bytes(1, C.byref(few), 2, 2, 16, 0, C.byref(fb), None) == 0
    assert fb.value > 0
    assert fwd(win=C.byref(few), ws=p, n=fb.value - 1) == 4
    assert lib.ngt_packed_workspace_bytes(1, w, 2, 2, 16, 256, None, None) == 1
    bwd = lambda **o: lib.ngt_packed_bwd(1, p, p, p, 32, 32, 32, p, p, p, w, 2, 2, 16, 1.0,
                                         o.get("table"), o.get("nb", 0), o.get("ids"), None,
                                         o.get("gq", p), p, p, o.get("gt"), None, 0, None)
    assert bwd() == 4  # no workspace
    assert bwd(gq=None) == 1 and bwd(gt=p) == 1 and bwd(table=p, ids=p, nb=3) == 1
    assert lib.ngt_packed_buckets(w, p, 2, p, p, None) == 1
    assert lib.ngt_packed_buckets(w, None, 1, p, p, None) == 1


def test_python_refusals():
    for bad in ([[1, 2]], [1.5], [-1], [(1 << 28) + 1], [True]):
        with pytest.raises(ValueError):
            PackedWindows(bad, device="cuda:0")
    with pytest.raises(ValueError, match="key lengths"):
        PackedWindows([1, 2], [1], device="cuda:0")
    with pytest.raises(ValueError, match="GPU"):
        PackedWindows([1], device="cpu")
    with pytest.raises(TypeError, match="PackedWindows"):
        packed_attention(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), [1])


class _Plan(PackedWindows):
    """A plan without device memory: enough for the checks before a launch."""

    def __init__(self, ql, kl=None, causal=False):
        self.struct = _plan(ql, kl or ql, causal)[0]
        self.q_lengths, self.k_lengths = list(ql), list(kl or ql)
        self.device = torch.device("cuda", 0)
        self.causal = causal


def test_bucket_refusals():
    w = _Plan([3, 2], [4, 1])
    for ids, err in ((torch.zeros(14, dtype=torch.uint8), ValueError),  # on the CPU
                     ([torch.zeros(3, 4)], ValueError),
                     ([torch.zeros(3, 4), torch.zeros(1, 2)], ValueError)):
        with pytest.raises(err):
            w.pack_buckets(ids)


def test_call_refusals_in_python():
    w = _Plan([3, 2])
    t = torch.zeros(5, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        packed_attention(t, t, t, w)
    with pytest.raises(ValueError, match=r"rows, heads"):
        packed_attention(t[0], t, t, w)


def test_more_blocks_than_a_launch_takes_are_refused():
    """Plans of more rows than any test holds: the counts alone decide."""
    lib = _lib.load()
    p = 1 << 20
    st, _ = _plan([4096], [4096], 0)
    for i in range(3):
        st.n_items_q[i] = st.n_items_k[i] = 1 << 22
    assert lib.ngt_packed_fwd(1, p, p, p, 64, 64, 64, C.byref(st), 4, 4, 16, 1.0, None, 0, None, p,
                              None, None, None, 0, None) == 2
    assert b"one launch" in lib.ngt_last_error()
    wb = C.c_size_t()
    assert lib.ngt_packed_workspace_bytes(1, C.byref(st), 4, 4, 16, 0, None, C.byref(wb)) == 0
    assert lib.ngt_packed_bwd(1, p, p, p, 64, 64, 64, p, p, p, C.byref(st), 4, 4, 16, 1.0, None, 0,
                              None, None, p, p, p, None, p, wb.value, None) == 2
    assert b"one launch" in lib.ngt_last_error()
    few, _ = _plan([1], [200], 1)
    few.n_windows = 1 << 24
    assert lib.ngt_packed_fwd(1, p, p, p, 16, 16, 16, C.byref(few), 1, 1, 16, 1.0, None, 0, None, p,
                              None, None, None, 0, None) == 2
