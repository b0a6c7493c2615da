"""The float64 restatement of packed attention: against one window by hand,
against differences, and its empty rows."""
import torch

from oracle import packed as OP


def _inputs(q_len, k_len, H, hkv, d, buckets=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(q_len), H, d, generator=g, dtype=torch.float64)
    k, v = (torch.randn(sum(k_len), hkv, d, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.randn(buckets, H, generator=g, dtype=torch.float64) if buckets else None
    ids = (torch.randint(-1, buckets + 1, (sum(a * b for a, b in zip(q_len, k_len)),), generator=g)
           if buckets else None)
    return q, k, v, table, ids


def test_one_window_one_head_by_hand():
    q, k, v, _, _ = _inputs([3], [5], 1, 1, 4)
    p = torch.softmax(q[:, 0] @ k[:, 0].t() * 0.5, 1)
    assert torch.allclose(OP.attention(q, k, v, [3], [5])[:, 0], p @ v[:, 0], atol=1e-14)


def test_windows_do_not_see_each_other_and_groups_share_their_key_head():
    ql, kl = [2, 0, 3], [4, 2, 3]
    q, k, v, _, _ = _inputs(ql, kl, 4, 2, 8)
    out = OP.attention(q, k, v, ql, kl, causal=True)
    for h in range(4):
        s = q[2:, h] @ k[6:, h // 2].t() / 8 ** 0.5
        s = s.masked_fill(~torch.ones(3, 3, dtype=torch.bool).tril(), -torch.inf)
        assert torch.allclose(out[2:, h], torch.softmax(s, 1) @ v[6:, h // 2], atol=1e-14)


def test_rows_that_see_nothing_are_zero_and_give_no_gradient():
    ql, kl = [4, 2], [2, 0]  # causal: the first two queries are before every key
    q, k, v, _, _ = _inputs(ql, kl, 2, 2, 8)
    out, dq, dk, dv = OP.fwd_bwd(q, k, v, torch.ones_like(q), ql, kl, causal=True)
    assert out[:2].abs().max() == 0 and dq[:2].abs().max() == 0 and out[4:].abs().max() == 0
    assert out[2:4].abs().min() > 0 and torch.isfinite(dk).all() and torch.isfinite(dv).all()


def test_gradients_against_differences():
    ql, kl = [3, 1], [4, 2]
    q, k, v, table, ids = _inputs(ql, kl, 2, 1, 8, buckets=3, seed=2)
    leaves = tuple(t.requires_grad_() for t in (q, k, v, table))
    assert torch.autograd.gradcheck(
        lambda a, b, c, t: OP.attention(a, b, c, ql, kl, True, None, t, ids), leaves,
        eps=1e-6, atol=1e-7, rtol=1e-6)
