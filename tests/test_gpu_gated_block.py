"""A transformer block over packed windows and its training step, as the operators would
be used together: joint projections, norm_rotary, causal packed_attention with grouped
heads, output projection with its residual, gated_linear, the second half with its
residual; backward, clipping, an optimizer step; and its form for single tokens.

Every operator's results are checked against float64 from the inputs and output
gradients that it really got, within the bounds of its own roundings."""
import math

import pytest
import torch

from neutrongt_amd import (PackedWindows, Rotary, clip_gradients, gated_linear, linear_epilogue,
                           norm_rotary, packed_attention)
from neutrongt_amd.encoder import WindowGraphormer, window_step
from oracle import packed as OP
from oracle import rotary as OR
from tests.test_gpu_gated_linear import _check as check_gated
from tests.test_gpu_gated_linear import _ref as ref_gated
from tests.test_gpu_linear_epilogue import _check as check_linear
from tests.test_gpu_linear_epilogue import _ref as ref_linear

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HB = 2.0 ** -8


class Block(torch.nn.Module):
    def __init__(self, dim, heads, kv_heads, hidden, dev):
        super().__init__()
        self.heads, self.kv_heads, self.d = heads, kv_heads, dim // heads
        make = lambda *s: torch.nn.Parameter((torch.randn(*s, device=dev) / math.sqrt(dim)).to(BF16))
        self.qkv, self.o = make((heads + 2 * kv_heads) * self.d, dim), make(dim, dim)
        self.gate, self.up, self.down = make(hidden, dim), make(hidden, dim), make(dim, hidden)
        self.q_gain, self.k_gain = (torch.nn.Parameter(1 + 0.1 * torch.randn(self.d, device=dev))
                                    for _ in range(2))
        self.rotary = Rotary(self.d // 2, device=dev)

    def rows(self, x, positions, keep=lambda name, t: t):
        """(q, k, v) of rows x at their positions."""
        h, hk = self.heads, self.kv_heads
        joint = keep("joint", linear_epilogue(x, self.qkv).view(-1, h + 2 * hk, self.d))
        q, k = norm_rotary(joint[:, :h], joint[:, h:h + hk], positions, self.rotary, self.q_gain,
                           self.k_gain)
        return keep("q", q), keep("k", k), keep("v", joint[:, h + hk:])

    def rest(self, x, q, k, v, win, keep=lambda name, t: t):
        a = keep("a", packed_attention(q, k, v, win))
        x = keep("x2", linear_epilogue(a.reshape(x.shape), self.o, residual=x))
        u = keep("u", gated_linear(x, self.gate, self.up))
        return linear_epilogue(u, self.down, residual=x)

    def forward(self, x, win, positions, keep=lambda name, t: t):
        return self.rest(x, *self.rows(x, positions, keep), win, keep)


def _setup(dev, lengths, seed):
    torch.manual_seed(seed)
    block = Block(64, 4, 2, 160, dev)
    win = PackedWindows(lengths, causal=True, device=dev)
    x, gy = (torch.randn(sum(lengths), 64).to(BF16).to(dev) for _ in range(2))
    return block, win, win.positions(), x, gy


def test_positions(dev):
    win = PackedWindows([3, 0, 1, 2], [3, 4, 9, 1], device=dev)
    assert win.positions().tolist() == [0, 1, 2, 8, -1, 0]
    assert PackedWindows([], device=dev).positions().shape == (0,)


@pytest.mark.parametrize("lengths", [[37, 1, 90, 0, 64], [1], [300, 150]])
def test_block_forward_and_backward(dev, lengths):
    block, win, positions, x, gy = _setup(dev, lengths, sum(lengths))
    kept = {}

    def keep(name, t):
        t.retain_grad()
        kept[name] = t
        return t

    x.requires_grad_()
    y = block(x, win, positions, keep)
    y.backward(gy)
    val = {n: t.detach().cpu() for n, t in kept.items()}
    grad = {n: t.grad.cpu() for n, t in kept.items()}
    par = {n: p.detach().cpu() for n, p in block.named_parameters()}
    par_grad = {n: p.grad for n, p in block.named_parameters()}

    ref = ref_linear(val["u"], par["down"], None, val["x2"], gy.cpu(), None)
    check_linear([y.detach(), grad["u"], par_grad["down"]], ref, "down")
    ref = ref_gated(val["x2"], par["gate"], par["up"], None, None, grad["u"], "silu")
    check_gated([val["u"]], ref[:1], "gated")
    check_gated([par_grad["gate"], par_grad["up"]], ref[2:4], "gated weights")
    # x2's gradient: the gated layer's, rounded to bf16, and the residual's, added in bf16
    want = ref[1][0] + gy.cpu().double()
    bound = ref[1][1] + HB * (want.abs() + ref[1][1])
    assert ((grad["x2"].double() - want).abs() <= bound).all()

    ref, bound = OP.bounds(val["q"], val["k"], val["v"], grad["a"], lengths, lengths, HB, causal=True)
    for name, got, r, b in zip(("out", "dq", "dk", "dv"), (val["a"], *(grad[c] for c in "qkv")), ref,
                               bound):
        over = ((got.double() - r).abs() - b).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"

    f, pos = block.rotary.frequencies, positions.cpu()
    for c, part in (("q", slice(0, 4)), ("k", slice(4, 6))):
        (r, b), (dr, db), (gr, gb) = OR.bounds(val["joint"][:, part], par[c + "_gain"], pos, f, "half",
                                               1.0, 1e-6, grad[c], HB, 2.0 ** -24)
        assert ((val[c].double() - r).abs() <= b).all()
        assert ((grad["joint"][:, part].double() - dr).abs() <= db).all()
        assert ((par_grad[c + "_gain"].double().cpu() - gr).abs() <= gb).all()
    assert torch.equal(grad["joint"][:, 6:], grad["v"])
    assert x.grad is not None and torch.isfinite(x.grad).all()


def test_captured_training_step(dev):
    """Forward, backward and clipping in a graph; every replay, with eager steps in
    between, gives the eager step's bits for the inputs of that replay."""
    block, win, positions, x, gy = _setup(dev, [40, 9, 128], 3)
    leaves = list(block.parameters())
    into = [torch.empty_like(p, dtype=torch.float32) for p in leaves]

    def step(into):
        y = block(x, win, positions)
        for p, g in zip(leaves, torch.autograd.grad(y, leaves, gy)):
            p.grad = g
        norm = clip_gradients(leaves, 1.0, out=into)
        return [y.detach(), norm, *into]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(into)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(into)
    for i in range(4):
        x.normal_()
        gy.normal_()
        want = [t.clone() for t in step([torch.empty_like(t) for t in into])]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want)), i
        size = math.sqrt(sum(float((t.double() ** 2).sum()) for t in into))
        assert abs(size - min(1.0, want[1].item())) <= 1e-6


def test_single_tokens_against_their_cached_keys(dev):
    """The last row of each window, its keys cached: the same bits as in the whole
    windows for what is computed by rows, and close to it behind the attention."""
    lengths = [37, 5, 130]
    block, win, positions, x, _ = _setup(dev, lengths, 6)
    with torch.no_grad():
        q, k, v = block.rows(x, positions)
        whole = block.rest(x, q, k, v, win)
        last = torch.tensor([36, 41, 171], device=dev)
        one = PackedWindows([1] * 3, lengths, causal=True, device=dev)
        q1, k1, v1 = block.rows(x[last], one.positions())
        # a projection of three rows takes another form than one of all of them
        for a, b in ((q1, q), (k1, k), (v1, v)):
            assert (a.float() - b[last].float()).abs().max() <= 4 * HB * b.float().abs().max()
        y = block.rest(x[last], q[last], k, v, one)
    assert (y.float() - whole[last].float()).abs().max() <= 16 * HB * whole.float().abs().max()


def test_training_step_clips(dev):
    """window_step with max_grad_norm: an SGD step from clipped gradients has the length
    lr * max_grad_norm; without it, and below the limit, the step is as it was."""
    torch.manual_seed(0)
    n, e = 200, 1000
    edges = torch.randint(0, n, (2, e), device=dev)
    edges = torch.cat([edges, torch.arange(n, device=dev).repeat(2, 1)], 1)
    x, labels = torch.randn(n, 20, device=dev), torch.randint(0, 5, (n,), device=dev)
    mask = torch.rand(n, device=dev) < 0.5

    def moved(limit):
        torch.manual_seed(1)
        model = WindowGraphormer(2, 4, 20, 32, 5).to(dev)
        before = [p.detach().clone() for p in model.parameters()]
        opt = torch.optim.SGD(model.parameters(), lr=0.5)
        window_step(model, opt, x, edges, labels, mask, autocast_dtype=BF16, max_grad_norm=limit)
        return [b - p.detach() for b, p in zip(before, model.parameters())]

    free, clipped, loose = moved(None), moved(1e-2), moved(1e6)
    size = math.sqrt(sum(float((t.double() ** 2).sum()) for t in clipped))
    assert abs(size - 0.5e-2) <= 1e-3 * 0.5e-2
    assert all(torch.equal(a, b) for a, b in zip(free, loose))
    assert math.sqrt(sum(float((t.double() ** 2).sum()) for t in free)) > 2 * size
