"""gated_linear's backward in every width of its products' blocks, the contraction whole and
in parts, against float64 (tests/test_gated_bwd_tiles.py says which size takes which)."""
import pytest
import torch

from tests.test_gated_bwd_tiles import SIZES
from tests.test_gpu_gated_linear import BF16, F32, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w_type", [BF16, F32])
@pytest.mark.parametrize("M,N,K", list(SIZES))
def test_gradients_in_every_width(dev, M, N, K, w_type):
    _case(dev, M, N, K, "silu", bias=w_type == F32, w_type=w_type, seed=M + K)
