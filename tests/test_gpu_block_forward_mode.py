"""Forward-mode differentiation is refused by norm_rotary and gated_linear, whichever
input carries the tangent and whether or not gradients are being recorded."""
import pytest
import torch

from neutrongt_amd import Rotary, gated_linear, norm_rotary
from tests.test_gpu_forward_mode import _refused, node  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(4))
def test_norm_rotary(dev, node, grad, which):  # noqa: F811
    rot, pos = Rotary(8, device=dev), torch.arange(5, device=dev)
    tensors = [torch.randn(s, device=dev) for s in ((5, 4, 8), (5, 2, 8), (8,), (8,))]
    if grad:  # another input than the one with the tangent
        tensors[(which + 1) % 4].requires_grad_()
    _refused(lambda q, k, a, b: norm_rotary(q, k, pos, rot, a, b), tensors, which)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(5))
def test_gated_linear(dev, node, grad, which):  # noqa: F811
    tensors = [torch.randn(s, device=dev).to(torch.bfloat16) for s in ((4, 8), (6, 8), (6, 8), (6,), (6,))]
    if grad:
        tensors[(which + 1) % 5].requires_grad_()
    _refused(lambda x, a, b, c, d: gated_linear(x, a, b, c, d), tensors, which)
