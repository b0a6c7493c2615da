"""The packed-window operators as one block of a graph transformer over a batch of
graphs, as they would be used: LayerNorm, joint projection, attention with a bias
per hop-distance bucket, output projection with its residual, LayerNorm, and the
two-layer FFN with GELU and residual; forward and backward under bf16 autocast.

Every operator's results are checked against float64 from the inputs and output
gradients that it really got, within the bounds of its own roundings (those of
test_gpu_packed and test_gpu_linear_epilogue); the LayerNorm's input gradient,
added to the residual's, closes the chain."""
import pytest
import torch

from neutrongt_amd import PackedWindows, linear_epilogue, packed_attention
from neutrongt_amd.layernorm import FusedLayerNorm
from neutrongt_amd.linear import WgradLinear, project
from oracle import packed as OP
from tests.test_gpu_linear_epilogue import HB, U, _check, _ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Block(torch.nn.Module):
    def __init__(self, dim, heads, buckets, hidden):
        super().__init__()
        self.heads = heads
        self.norm1, self.norm2 = (FusedLayerNorm(dim, out_bf16=True) for _ in range(2))
        self.q, self.k, self.v = (WgradLinear(dim, dim) for _ in range(3))
        self.o = torch.nn.Linear(dim, dim)
        self.up, self.down = torch.nn.Linear(dim, hidden), torch.nn.Linear(hidden, dim)
        self.table = torch.nn.Parameter(torch.randn(buckets, heads))

    def forward(self, x, win, ids, keep=lambda name, t: t):
        n, dim = x.shape
        shape = (n, self.heads, dim // self.heads)
        qkv = project(keep("h", self.norm1(x)), self.q, self.k, self.v)
        q, k, v = (keep(c, t.view(shape)) for c, t in zip("qkv", qkv))
        table = keep("table", self.table.to(q.dtype))
        a = keep("a", packed_attention(q, k, v, win, bias_table=table, buckets=ids))
        x = keep("x2", linear_epilogue(a.view(n, dim), self.o.weight, self.o.bias, residual=x))
        h = keep("h2", self.norm2(x))
        u = keep("u", linear_epilogue(h, self.up.weight, self.up.bias, "gelu"))
        return linear_epilogue(u, self.down.weight, self.down.bias, residual=x)


def _setup(dev, lengths, seed):
    torch.manual_seed(seed)
    block = Block(64, 4, 11, 160).to(dev)
    x = torch.randn(sum(lengths), 64).to(BF16)
    ids = torch.randint(0, 11, (sum(n * n for n in lengths),))
    ids[torch.rand(ids.numel()) < 0.05] = 255
    win = PackedWindows(lengths, device=dev)
    return block, x, torch.randn(sum(lengths), 64).to(BF16), ids, win, win.pack_buckets(ids.to(dev))


@pytest.mark.parametrize("lengths", [[37, 1, 90, 0, 64], [1], [300, 150]])
def test_block_forward_and_backward(dev, lengths):
    block, x, gy, ids, win, packed = _setup(dev, lengths, sum(lengths))
    kept = {}

    def keep(name, t):
        t.retain_grad()
        kept[name] = t
        return t

    xd = x.to(dev).requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        y = block(xd, win, packed, keep)
    y.backward(gy.to(dev))
    val = {n: t.detach().cpu() for n, t in kept.items()}
    grad = {n: t.grad.cpu() for n, t in kept.items()}

    def linear(layer, x_in, res, out, g_out, g_in, act):
        w, b = (t.detach().cpu().to(BF16) for t in (layer.weight, layer.bias))
        got = [out, g_in, layer.weight.grad, layer.bias.grad]
        _check(got, _ref(x_in, w, b, res, g_out, act, torch.float32), "block")

    linear(block.down, val["u"], val["x2"], y.detach(), gy, grad["u"], None)
    linear(block.up, val["h2"], None, kept["u"].detach(), grad["u"], grad["h2"], "gelu")
    a2, ga = (t.reshape(-1, 64) for t in (val["a"], grad["a"]))
    linear(block.o, a2, x, kept["x2"].detach(), grad["x2"], ga, None)

    ref, bound = OP.bounds(val["q"], val["k"], val["v"], grad["a"], lengths, lengths, 2.0 ** -8,
                           table=val["table"], ids=ids)
    for name, got, r, b in zip(("out", "dq", "dk", "dv", "dtable"),
                               (val["a"], *(grad[c] for c in "qkv"), grad["table"]), ref, bound):
        over = ((got.double() - r).abs() - b).max().item()
        assert over <= 0, f"{name}: {over:.3e} over the bound"

    # x2's gradient: the residual's, which is gy, and norm2's in bf16, added in bf16.
    # The norm's: each fp32 step off by u of its operands, 64-term sums by 64 u, and
    # xhat by as much of |x| rstd: below 1024 u of the terms' absolute values
    x2, g = val["x2"].double(), grad["h2"].double() * block.norm2.weight.detach().double().cpu()
    rstd = 1 / (x2.var(1, unbiased=False, keepdim=True) + block.norm2.eps).sqrt()
    hat = (x2 - x2.mean(1, keepdim=True)) * rstd
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    mag = rstd * (g.abs() + g.abs().mean(1, keepdim=True)
                  + (1 + hat.abs()) * (g * hat).abs().mean(1, keepdim=True)
                  + (1 + hat.abs()) * g.abs().mean(1, keepdim=True))
    e = 1024 * U * mag
    e = e + HB * (dx.abs() + e)
    want = dx + gy.double()
    e = e + HB * (want.abs() + e)
    assert ((grad["x2"].double() - want).abs() <= e).all()
    assert xd.grad is not None and torch.isfinite(xd.grad).all()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())


def test_captured_block_step(dev):
    """Forward and backward of the block in a graph; every replay, with eager steps in
    between, gives the eager step's bits for the inputs of that replay."""
    block, x, gy, _, win, packed = _setup(dev, [40, 9, 128], 3)
    xd, g = x.to(dev).requires_grad_(), gy.to(dev)
    leaves = [xd, *block.parameters()]

    def step():
        with torch.autocast("cuda", dtype=BF16, cache_enabled=False):
            y = block(xd, win, packed)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(4):
        with torch.no_grad():
            xd.normal_()
            g.normal_()
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want)), i


def test_inference_of_the_block_gives_the_training_forward(dev):
    block, x, _, _, win, packed = _setup(dev, [200, 3, 55], 4)
    with torch.autocast("cuda", dtype=BF16):
        y = block(x.to(dev).requires_grad_(), win, packed)
        with torch.no_grad():
            assert torch.equal(block(x.to(dev), win, packed), y)
