"""Single tokens beside whole packed windows (tests/test_gpu_gated_block.py): what is computed
by rows has the same bits, however many rows a call has and wherever they lie."""
import pytest
import torch

from neutrongt_amd import PackedWindows, norm_rotary
from tests.test_gpu_gated_block import HB, _setup

pytestmark = pytest.mark.gpu


def test_single_tokens_by_rows(dev):
    lengths = [37, 5, 130]
    block, win, positions, x, _ = _setup(dev, lengths, 6)
    kept = {}
    with torch.no_grad():
        q, k, v = block.rows(x, positions, lambda name, t: kept.setdefault(name, t))
        last = torch.tensor([36, 41, 171], device=dev)
        one = PackedWindows([1] * 3, lengths, causal=True, device=dev)
        assert one.positions().tolist() == [36, 4, 129]
        joint = kept["joint"][last]
        h, hk = block.heads, block.kv_heads
        q1, k1 = norm_rotary(joint[:, :h], joint[:, h:h + hk], one.positions(), block.rotary,
                             block.q_gain, block.k_gain)
        assert torch.equal(q1, q[last]) and torch.equal(k1, k[last])
        # at the neighbouring positions neither has
        for off in (-1, 1):
            q2, k2 = norm_rotary(joint[:, :h], joint[:, h:h + hk], one.positions() + off, block.rotary,
                                 block.q_gain, block.k_gain)
            assert not torch.equal(q2, q[last]) and not torch.equal(k2, k[last])
        # and these, their keys in the cached rows, give what the whole windows give
        cached_k, cached_v = k.clone(), v.clone()
        cached_k[last], cached_v[last] = k1, joint[:, h + hk:]
        assert torch.equal(cached_k, k) and torch.equal(cached_v, v)
        y = block.rest(x[last], q1, cached_k, cached_v, one)
        whole = block.rest(x, q, k, v, win)
    assert (y.float() - whole[last].float()).abs().max() <= 16 * HB * whole.float().abs().max()
