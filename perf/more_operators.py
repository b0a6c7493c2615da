"""Performance cases of the operators around packed attention in a transformer
block and its training step: norm and rotation of queries and keys by head, the
gated linear layer, and the clipping of gradients by their global norm.

A case is a dict of plain values; ``prepare`` builds what a program holds
before the call, ``run`` is one pass (the framework's kernels where ``own`` is
true, else the plain form in 32 bits), ``work`` the bytes and operations that
pass cannot do without, ``exact`` its outputs from the definition in 64 bits.

Families
  rotary  RMS norm of each query and key head with a gain, and the rotation of
          its first components by the row's position; forward, or forward and
          backward
  gated   act(x Wg^T + bg) * (x Wu^T + bu); forward, or forward and backward
  clip    the 2-norm over a model's gradients, and the gradients scaled down to
          a largest norm
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def _rotary(name, rows, heads, kv_heads, dim, rotated, layout, norm, far, factor, dtype, train):
    c = dict(kind="rotary", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rotated=rotated,
             layout=layout, norm=norm, far=far, factor=factor, dtype=dtype, train=train)
    return dict(c, name=name) if name else c


def _gated(name, rows, n_in, n_out, act, bias, train):
    c = dict(kind="gated", rows=rows, n_in=n_in, n_out=n_out, act=act, bias=bias, dtype="bf16",
             train=train)
    return dict(c, name=name) if name else c


def _clip(name, layers, hidden, ffn, classes, dtype, out, above):
    c = dict(kind="clip", layers=layers, hidden=hidden, ffn=ffn, classes=classes, dtype=dtype,
             out=out, above=above)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of each of a few requests, far into their contexts: latency
        _rotary("rotary_tokens_bf16", 16, 32, 8, 128, 128, "half", True, 131072, 8.0, "bf16", False),
        # the prompts of a server
        _rotary("rotary_prompt_bf16", 12289, 32, 8, 128, 128, "half", True, 0, 1.0, "bf16", False),
        # the large preset (32 heads of 24) over a whole window, trained
        _rotary("rotary_large_train_bf16", 32768, 32, 32, 24, 24, "interleaved", True, 0, 1.0,
                "bf16", True),
        # fp32 training, half of each head rotated, positions stretched fourfold, no norm
        _rotary("rotary_part_train_f32", 10007, 16, 4, 64, 32, "half", False, 0, 4.0, "f32", True),
        # a few served nodes through the preset's width: latency
        _gated("gated_nodes_bf16", 5, 768, 768, "gelu", True, False),
        # single tokens of many requests: the weights' bytes
        _gated("gated_tokens_bf16", 33, 2048, 8192, "silu", False, False),
        # a wide feed-forward block over a ragged number of rows
        _gated("gated_wide_bf16", 10007, 1024, 4096, "silu", False, False),
        # the large preset's width over a whole window, trained
        _gated("gated_window_train_bf16", 32768, 768, 2048, "silu", True, True),
        # the slim preset's many small gradients: latency
        _clip("clip_slim_f32", 4, 64, 64, 40, "f32", "f32", True),
        # the large preset's gradients
        _clip("clip_large_f32", 12, 768, 768, 47, "f32", "f32", True),
        # most steps of a training run: nothing to clip, in place
        _clip("clip_below_f32", 12, 768, 2048, 47, "f32", "", False),
        # a wide model's bf16 gradients, clipped into fp32 for the optimizer
        _clip("clip_wide_bf16", 24, 1024, 4096, 1001, "bf16", "f32", True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["rotary", "gated", "clip"])
    if kind == "rotary":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (8, 8, 8), (32, 32, 24), (16, 4, 64),
                                           (8, 8, 16), (12, 12, 80), (16, 2, 40), (8, 1, 256),
                                           (5, 5, 96)])
        rows = int(_log(rng, 1, 65536))
        while rows * (heads + kv_heads) * dim > 32768 * 64 * 24:
            rows = max(1, int(rows * 0.7))
        rotated = rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2 or 2])
        train = rng.random() < 0.5
        return _rotary(None, rows, heads, kv_heads, dim, rotated,
                       rng.choice(["half", "interleaved"]), rng.random() < 0.7,
                       0 if train else int(_log(rng, 1, 1 << 20)), rng.choice([1.0, 1.0, 4.0, 8.0]),
                       rng.choice(["bf16", "bf16", "f32"]), train)
    if kind == "gated":
        rows = int(_log(rng, 1, 32768))
        step = rng.choice([8, 8, 8, 1])
        n_in, n_out = (step * int(_log(rng, 64 // step, 8192 // step)) for _ in range(2))
        train = rng.random() < 0.5
        while (rows * n_in * n_out > 32768 * 768 * 2048 * (1 if train else 2)
               or rows * (n_in + n_out) > 32768 * 3000):
            rows = max(1, int(rows * 0.6))
        return _gated(None, rows, n_in, n_out, rng.choice(["silu", "silu", "gelu", "relu"]),
                      rng.random() < 0.4, train)
    hidden = 8 * int(_log(rng, 4, 128))
    ffn = hidden * rng.choice([1, 2, 4])
    layers = int(_log(rng, 1, 25))
    above = rng.random() < 0.7
    dtype = rng.choice(["f32", "f32", "bf16"])
    out = rng.choice([dtype, "f32"]) if above else ""
    return _clip(None, layers, hidden, ffn, int(_log(rng, 2, 1001)), dtype, out, above)


def _shapes(case):
    """The parameters of an encoder: projections, feed-forward halves, norms, input and readout."""
    h, f, c = case["hidden"], case["ffn"], case["classes"]
    layer = [(h, h), (h,)] * 4 + [(f, h), (f,), (h, f), (h,)] + [(h,)] * 4
    return [(h, 100), (h,)] + layer * case["layers"] + [(h,)] * 2 + [(c, h), (c,)]


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _positions(case, seed):
    """Windows back to back, each from position 0; or, far into their contexts, a row each."""
    n, rng = case["rows"], random.Random(int(seed) * 31 + 5)
    if case["far"]:
        return torch.tensor([rng.randrange(case["far"]) for _ in range(n)], dtype=torch.int32)
    out, left = [], n
    while left:
        m = min(left, int(_log(rng, 1, 8192)))
        out.append(torch.arange(m, dtype=torch.int32))
        left -= m
    return torch.cat(out)


def prepare(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]

    def normal(*shape, by=1.0, grad=False):
        t = (torch.randn(*shape, device=DEV, generator=g) * by).to(dt)
        return t.requires_grad_() if grad else t

    train = case.get("train", False)
    if case["kind"] == "gated":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        w = normal(2 * n, k, by=k ** -0.5)
        b = normal(2 * n, by=0.1) if case["bias"] else None
        leaves = dict(x=normal(m, k), wg=w[:n].clone(), wu=w[n:].clone())
        if b is not None:
            leaves.update(bg=b[:n].clone(), bu=b[n:].clone())
        for t in leaves.values():
            t.requires_grad_(train)
        return dict(case=case, leaves=leaves, gy=normal(m, n) if train else None)
    if case["kind"] == "clip":
        # layers of different scales; all gradients lie in one buffer, as the buckets of a
        # data-parallel program do, and so does what they are clipped into
        rng, shapes = random.Random(int(seed) * 13 + 1), _shapes(case)
        flat = torch.cat([normal(math.prod(s), by=1e-3 * _log(rng, 0.1, 10)) for s in shapes])
        flat_out = torch.empty_like(flat, dtype=_DT[case["out"]]) if case["out"] else None
        grads, out = (None if t is None else
                      [p.view(s) for p, s in zip(t.split([math.prod(s) for s in shapes]), shapes)]
                      for t in (flat, flat_out))
        # the norm's own size is known well enough to be on either side of it
        size = math.sqrt(sum(t.numel() for t in grads))
        st = dict(case=case, grads=grads, out=out, flat=flat, flat_out=flat_out,
                  max_norm=size * (1e-6 if case["above"] else 1.0))
        if own:
            st["params"] = [torch.nn.Parameter(torch.empty_like(t)) for t in grads]
            for p, t in zip(st["params"], grads):
                p.grad = t
        return st
    n, h, hkv, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    # queries, keys and values of one joint projection
    joint = normal(n, h + 2 * hkv, d)
    q, k = joint[:, :h].detach(), joint[:, h:h + hkv].detach()
    gains = [1 + 0.1 * torch.randn(d, device=DEV, generator=g) for _ in range(2)]
    st = dict(case=case, q=q, k=k, pos=_positions(case, seed).to(DEV),
              gains=gains if case["norm"] else [None, None],
              gq=normal(n, h, d) if train else None, gk=normal(n, hkv, d) if train else None)
    for t in (q, k, *st["gains"]):
        if t is not None:
            t.requires_grad_(train)
    if own:
        from neutrongt_amd import Rotary

        st["rotary"] = Rotary(case["rotated"], layout=case["layout"], scaling="linear",
                              factor=case["factor"], device=DEV)
    return st


# ------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from neutrongt_amd import clip_gradients, gated_linear, norm_rotary

    case = st["case"]
    if case["kind"] == "clip":
        norm = clip_gradients(st["params"], st["max_norm"], out=st["out"])
        return norm, st["flat"] if st["out"] is None else st["flat_out"]
    if case["kind"] == "gated":
        v = st["leaves"]
        if not case["train"]:
            with torch.no_grad():
                return gated_linear(v["x"], v["wg"], v["wu"], v.get("bg"), v.get("bu"),
                                    activation=case["act"])
        y = gated_linear(v["x"], v["wg"], v["wu"], v.get("bg"), v.get("bu"),
                         activation=case["act"])
        return (y.detach(), *torch.autograd.grad(y, list(v.values()), st["gy"]))
    args = (st["q"], st["k"], st["pos"], st["rotary"], *st["gains"])
    if not case["train"]:
        with torch.no_grad():
            return norm_rotary(*args, eps=EPS)
    yq, yk = norm_rotary(*args, eps=EPS)
    leaves = [t for t in (st["q"], st["k"], *st["gains"]) if t is not None]
    return (yq.detach(), yk.detach(),
            *torch.autograd.grad((yq, yk), leaves, (st["gq"], st["gk"])))


def _run_plain(st):
    with torch.no_grad():
        return {"clip": _plain_clip, "gated": _plain_gated, "rotary": _plain_rotary}[
            st["case"]["kind"]](st)


def _plain_clip(st):
    squares = torch.stack([(t.float() * t.float()).sum() for t in st["grads"]])
    norm = squares.double().sum().sqrt()
    by = torch.clamp(st["max_norm"] / norm, max=1.0).float()
    into = st["out"] or st["grads"]
    for t, o in zip(st["grads"], into):
        o.copy_((t.float() * by).to(o.dtype))
    return norm.float(), st["flat"] if st["out"] is None else st["flat_out"]


def _plain_gated(st):
    case, dt = st["case"], st["leaves"]["x"].dtype
    v = {n: t.float() for n, t in st["leaves"].items()}
    a, u = v["x"] @ v["wg"].t(), v["x"] @ v["wu"].t()
    if case["bias"]:
        a, u = a + v["bg"], u + v["bu"]
    if case["act"] == "silu":
        s = 1 / (1 + torch.exp(-a))
        act, slope = a * s, s * (1 + a * (1 - s))
    elif case["act"] == "gelu":
        cdf = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        act, slope = a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    else:
        slope = (a > 0).float()
        act = a * slope
    y = (act * u).to(dt)
    if not case["train"]:
        return y
    gy = st["gy"].float()
    da, du = gy * u * slope, gy * act
    out = [y, da @ v["wg"] + du @ v["wu"], da.t() @ v["x"], du.t() @ v["x"]]
    if case["bias"]:
        out += [da.sum(0), du.sum(0)]
    return tuple(t.to(dt) for t in out)


def _angles(case, pos):
    """cos and sin [rows, 1, rotated / 2], the angles in 64 bits."""
    r = case["rotated"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r) / case["factor"]
    t = pos.double()[:, None] * f
    return torch.cos(t)[:, None].float(), torch.sin(t)[:, None].float()


def _pairs(case):
    r = case["rotated"]
    if case["layout"] == "half":
        return slice(0, r // 2), slice(r // 2, r)
    return slice(0, r, 2), slice(1, r, 2)


def _rotated(case, u, cos, sin):
    a, b = _pairs(case)
    y = u.clone()
    y[..., a] = u[..., a] * cos - u[..., b] * sin
    y[..., b] = u[..., a] * sin + u[..., b] * cos
    return y


def _plain_rotary(st):
    case = st["case"]
    cos, sin = _angles(case, st["pos"])
    ys, dxs, dgains = [], [], []
    for x, gain, gy in zip((st["q"], st["k"]), st["gains"], (st["gq"], st["gk"])):
        u, dt = x.float(), x.dtype
        if case["norm"]:
            by = 1 / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS)
            hat = u * by
            u = hat * gain
        ys.append(_rotated(case, u, cos, sin).to(dt))
        if not case["train"]:
            continue
        g = _rotated(case, gy.float(), cos, -sin)
        if case["norm"]:
            dgains.append((g * hat).sum(1).double().sum(0).to(gain.dtype))
            g = g * gain
            g = (g - hat * (g * hat).mean(-1, keepdim=True)) * by
        dxs.append(g.to(dt))
    return (*ys, *dxs, *dgains)


# ----------------------------------------------------------- work and the truth
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        out = {"": 0, "f32": 4, "bf16": 2}[case["out"]]
        return {"bytes": n * (es + out) + 4, "flops": n * (3 if case["out"] else 2)}
    if case["kind"] == "gated":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        params = 2 * n * (k + (1 if case["bias"] else 0))
        byte = es * (m * k + params + m * n)
        if case["train"]:
            byte += es * (m * n + m * k + params)
        return {"bytes": byte, "flops": 4 * m * n * k * (3 if case["train"] else 1)}
    n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    byte = es * n * (4 if case["train"] else 2) + 4 * case["rows"]
    gains = 8 * case["dim"] if case["norm"] else 0
    return {"bytes": byte + gains * (2 if case["train"] else 1),
            "flops": n * (8 if case["train"] else 3) + n * (
                (10 if case["train"] else 4) if case["norm"] else 0)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "clip":
        big = st["flat"].double()
        norm = torch.sqrt(torch.dot(big, big))
        return norm, big * min(1.0, st["max_norm"] / float(norm))
    if case["kind"] == "gated":
        v = {n: t.detach().double().requires_grad_(case["train"])
             for n, t in st["leaves"].items()}
        f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "relu": torch.relu}[case["act"]]
        y = f(torch.nn.functional.linear(v["x"], v["wg"], v.get("bg"))) * (
            torch.nn.functional.linear(v["x"], v["wu"], v.get("bu")))
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, list(v.values()), st["gy"].double()))
    leaf = [t.detach().double().requires_grad_(case["train"])
            for t in (st["q"], st["k"], *st["gains"]) if t is not None]
    r, half = case["rotated"], case["rotated"] // 2
    angle = st["pos"].double()[:, None] / case["factor"] * torch.tensor(
        [10000.0 ** (-2 * i / r) for i in range(half)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    ys = []
    for i, x in enumerate(leaf[:2]):
        if case["norm"]:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * leaf[2 + i]
        front = x[..., :r]
        pair = (front.unflatten(-1, (2, half)).transpose(-1, -2) if case["layout"] == "half"
                else front.unflatten(-1, (half, 2)))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.transpose(-1, -2) if case["layout"] == "half" else z
        ys.append(torch.cat([z.flatten(-2), x[..., r:]], -1))
    if not case["train"]:
        return tuple(ys)
    return (*(y.detach() for y in ys),
            *torch.autograd.grad(ys, leaf, (st["gq"].double(), st["gk"].double())))
