"""Forward-mode differentiation is refused by the packed attention and the linear
epilogue, whichever input carries the tangent and whether or not gradients are being
recorded: never a result whose tangent is silently gone."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from neutrongt_amd import PackedWindows, _lib, linear_epilogue, packed_attention

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(params=["cpp", "python"])
def node(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "node_ext", lambda: None)
    else:
        assert _lib.autograd_ext() is not None


def _refused(call, tensors, which):
    with fw.dual_level():
        given = [fw.make_dual(t, torch.ones_like(t)) if i == which else t
                 for i, t in enumerate(tensors)]
        with pytest.raises((NotImplementedError, RuntimeError)):
            call(*given)
    with fw.dual_level(), torch.no_grad():
        given = [fw.make_dual(t, torch.ones_like(t)) if i == which else t
                 for i, t in enumerate(tensors)]
        with pytest.raises((NotImplementedError, RuntimeError)):
            call(*given)
    call(*tensors)  # outside of forward mode the same tensors are taken


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(4))
def test_packed_attention(dev, node, dtype, grad, which):
    win = PackedWindows([5, 3], device=dev)
    ids = win.pack_buckets(torch.zeros(34, dtype=torch.uint8, device=dev))
    shapes = [(8, 4, 16), (8, 2, 16), (8, 2, 16), (3, 4)]
    tensors = [torch.randn(s, device=dev).to(dtype) for s in shapes]
    if grad:  # another input than the one with the tangent
        tensors[(which + 1) % 4].requires_grad_()
    _refused(lambda q, k, v, t: packed_attention(q, k, v, win, bias_table=t, buckets=ids), tensors,
             which)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(4))
def test_linear_epilogue(dev, node, act, grad, which):
    shapes = [(4, 8), (6, 8), (6,), (4, 6)]
    tensors = [torch.randn(s, device=dev).to(BF16) for s in shapes]
    if grad:
        tensors[(which + 1) % 4].requires_grad_()
    _refused(lambda x, w, b, r: linear_epilogue(x, w, b, act, r), tensors, which)
