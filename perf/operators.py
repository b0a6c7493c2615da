"""Performance cases of the packed-window operators: attention over windows of
different lengths (grouped heads, causal order, single-node queries), the bias
learned per pair bucket in it, and the linear layer with its epilogue.

A case is a dict of plain values; ``prepare`` builds what a program holds
before the call, ``run`` is one pass (the framework's kernels where ``own`` is
true, else the plain form in 32 bits), ``work`` the bytes and operations that
pass cannot do without, ``exact`` its outputs from the definition in 64 bits.

Families
  attn    attention over packed windows, forward (serving) or forward and
          backward (training), without a bias
  bias    the same with a learned bias per pair bucket, whose gradient is
          returned too; one pair in about thirty is not attended
  nodes   a few query rows per window against its cached keys
  linear  act(x W^T + b) + residual, forward or forward and backward
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
NOT_ATTENDED = 255
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def _attn(name, windows, shortest, longest, heads, kv_heads, dim, dtype, causal, train):
    c = dict(kind="attn", windows=windows, shortest=shortest, longest=longest, heads=heads,
             kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal, train=train)
    return dict(c, name=name) if name else c


def _bias(name, windows, shortest, longest, heads, dim, dtype, buckets, train):
    c = dict(kind="bias", windows=windows, shortest=shortest, longest=longest, heads=heads,
             kv_heads=heads, dim=dim, dtype=dtype, causal=False, train=train, buckets=buckets)
    return dict(c, name=name) if name else c


def _nodes(name, windows, shortest, longest, rows, heads, kv_heads, dim, dtype):
    c = dict(kind="nodes", windows=windows, shortest=shortest, longest=longest, rows=rows,
             heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=True, train=False)
    return dict(c, name=name) if name else c


def _linear(name, rows, n_in, n_out, act, residual, train):
    c = dict(kind="linear", rows=rows, n_in=n_in, n_out=n_out, act=act, residual=residual,
             dtype="bf16", train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the windows of a partitioned citation graph, trained with the slim preset's 8 heads of 8
        _attn("attn_slim_train_bf16", 24, 100, 1500, 8, 8, 8, "bf16", False, True),
        # grouped heads over sequences of different lengths in causal order: training ...
        _attn("attn_causal_train_bf16", 6, 200, 4096, 16, 4, 64, "bf16", True, True),
        # ... and the forward pass of a server over whole prompts
        _attn("attn_prompt_bf16", 5, 500, 4096, 32, 8, 128, "bf16", True, False),
        # fp32 training with heads of 16, ragged windows
        _attn("attn_train_f32", 9, 33, 1777, 8, 8, 16, "f32", False, True),
        # single nodes against short cached windows: latency
        _nodes("nodes_small_bf16", 8, 60, 1000, 1, 8, 8, 16, "bf16"),
        # single tokens of many requests against long caches
        _nodes("nodes_long_bf16", 32, 1000, 16384, 1, 32, 8, 128, "bf16"),
        # the slim preset with structural encodings: hop-distance buckets over one window, fp32
        _bias("bias_slim_f32", 1, 3001, 3001, 8, 8, "f32", 40, True),
        # the large preset (32 heads of 24) over a few windows, bf16 training
        _bias("bias_large_bf16", 3, 1000, 3333, 32, 24, "bf16", 64, True),
        # evaluation of many small graphs in one call
        _bias("bias_graphs_eval_bf16", 300, 8, 200, 8, 64, "bf16", 21, False),
        # a few served nodes through one projection: latency
        _linear("linear_nodes_bf16", 5, 768, 768, "gelu", True, False),
        # the large preset's FFN half-step over a whole window, trained
        _linear("linear_window_bf16", 32768, 768, 768, "gelu", True, True),
        # a wide feed-forward projection over a ragged number of rows
        _linear("linear_wide_bf16", 10007, 1024, 4096, "gelu", False, False),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choices(["attn", "bias", "nodes", "linear"], [4, 3, 2, 3])[0]
    if kind == "linear":
        rows = int(_log(rng, 1, 32768))
        n_in, n_out = (8 * int(_log(rng, 8, 512)) for _ in range(2))
        while rows * n_in * n_out > 10007 * 1024 * 4096 or rows * n_out > 32768 * 1024:
            rows = max(1, int(rows * 0.6))
        return _linear(None, rows, n_in, n_out, rng.choice(["none", "relu", "gelu"]),
                       rng.random() < 0.5, rng.random() < 0.5)
    windows = int(_log(rng, 1, 64))
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "nodes":
        heads, kv_heads, dim = rng.choice([(8, 8, 16), (32, 8, 128), (16, 4, 64), (8, 1, 64),
                                           (32, 32, 24), (12, 12, 32)])
        rows = rng.choice([1, 1, 1, 2, 4])
        longest = int(_log(rng, 50, 16384))
        while windows * longest * kv_heads * dim > 32 * 16384 * 8 * 128:
            longest //= 2
        return _nodes(None, windows, max(1, longest // 8), longest, rows, heads, kv_heads, dim,
                      dtype)
    heads, kv_heads, dim = rng.choice([(8, 8, 8), (8, 8, 16), (32, 32, 24), (8, 8, 32), (8, 8, 64),
                                       (16, 4, 64), (16, 2, 40), (16, 4, 128)])
    longest = int(_log(rng, 16, 4096))
    # a padded batch of all heads' scores stays below the largest listed case's
    room = 3 * 3333 ** 2 * 32 if kind == "bias" else 5 * 4096 ** 2 * 32
    work = 5 * 4096 ** 2 * 32 * 128 // 4
    while (windows * longest ** 2 * heads > room or windows * longest ** 2 * heads * dim > work):
        windows, longest = max(1, int(windows * 0.8)), max(16, int(longest * 0.9))
    shortest = max(1, longest // rng.choice([1, 4, 16]))
    train = rng.random() < 0.6
    if kind == "bias":
        return _bias(None, windows, shortest, longest, heads, dim, dtype,
                     int(_log(rng, 8, 200)), train)
    return _attn(None, windows, shortest, longest, heads, kv_heads, dim, dtype,
                 rng.random() < 0.5, train)


def _lengths(case):
    """The windows' key lengths: the longest first, the others spread over the
    logarithm of the range; the same for every seed, so that ``work`` knows them."""
    w, lo, hi = case["windows"], case["shortest"], case["longest"]
    rng = random.Random(w * 1000003 + lo * 1009 + hi)
    return [hi] + [min(hi, int(_log(rng, lo, hi + 1))) for _ in range(w - 1)]


def _both_lengths(case):
    nk = _lengths(case)
    return [min(case["rows"], n) for n in nk] if case["kind"] == "nodes" else nk, nk


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths))]


def _padded_rows(lengths):
    """[W, longest] row of each place of a padded batch, and whether it is one."""
    at = torch.arange(max(lengths), device=DEV)
    n = torch.tensor(lengths, device=DEV)
    start = torch.tensor(_starts(lengths), device=DEV)
    there = at < n[:, None]
    return torch.where(there, start[:, None] + at, 0), there


def prepare(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]

    def normal(*shape, by=1.0, grad=False):
        t = (torch.randn(*shape, device=DEV, generator=g) * by).to(dt)
        return t.requires_grad_() if grad and case["train"] else t

    if case["kind"] == "linear":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        return dict(case=case, x=normal(m, k, grad=True), w=normal(n, k, by=k ** -0.5, grad=True),
                    b=normal(n, by=0.1, grad=True),
                    r=normal(m, n) if case["residual"] else None,
                    gy=normal(m, n) if case["train"] else None)
    nq, nk = _both_lengths(case)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    st = dict(case=case, nq=nq, nk=nk, q=normal(sum(nq), h, d, grad=True),
              k=normal(sum(nk), hkv, d, grad=True), v=normal(sum(nk), hkv, d, grad=True),
              go=normal(sum(nq), h, d) if case["train"] else None, rows_q=_padded_rows(nq),
              rows_k=_padded_rows(nk), ids=None, table=None)
    if case["kind"] == "bias":
        b = case["buckets"]
        st["table"] = normal(b, h, by=0.5, grad=True)
        # hop distances between nodes placed at random, the nearest buckets the fullest
        ids = []
        for n in nk:
            at = torch.rand(n, device=DEV, generator=g)
            far = (at[:, None] - at[None, :]).abs().sqrt() * (b - 1)
            far = (far + torch.rand(n, n, device=DEV, generator=g)).to(torch.uint8)
            cut = torch.rand(n, n, device=DEV, generator=g) < 1 / 32
            ids.append(torch.where(cut, NOT_ATTENDED, far).to(torch.uint8).flatten())
        st["ids"] = torch.cat(ids)
    if own:
        from neutrongt_amd import PackedWindows

        st["windows"] = PackedWindows(nq, nk, causal=case["causal"], device=DEV)
        st["buckets"] = (st["windows"].pack_buckets(st["ids"]) if st["ids"] is not None else None)
    else:
        st["pad_ids"] = _padded_ids(st) if st["ids"] is not None else None
    return st


def _padded_ids(st):
    """[W, longest, longest] ids of the padded batch (the plain form's layout of them)."""
    nk = st["nk"]
    out = torch.full((len(nk), max(nk), max(nk)), NOT_ATTENDED, dtype=torch.uint8, device=DEV)
    at = 0
    for w, n in enumerate(nk):
        out[w, :n, :n] = st["ids"][at:at + n * n].view(n, n)
        at += n * n
    return out


# ------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from neutrongt_amd import linear_epilogue, packed_attention

    case = st["case"]
    if case["kind"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        if not case["train"]:
            with torch.no_grad():
                return linear_epilogue(st["x"], st["w"], st["b"], activation=act, residual=st["r"])
        y = linear_epilogue(st["x"], st["w"], st["b"], activation=act, residual=st["r"])
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["gy"]))
    more = dict(bias_table=st["table"], buckets=st["buckets"]) if st["table"] is not None else {}
    if not case["train"]:
        with torch.no_grad():
            return packed_attention(st["q"], st["k"], st["v"], st["windows"], **more)
    out = packed_attention(st["q"], st["k"], st["v"], st["windows"], **more)
    leaves = [st["q"], st["k"], st["v"]] + ([st["table"]] if more else [])
    return (out.detach(), *torch.autograd.grad(out, leaves, st["go"]))


def _run_plain(st):
    with torch.no_grad():
        return _plain_linear(st) if st["case"]["kind"] == "linear" else _plain_attention(st)


def _plain_linear(st):
    case, dt = st["case"], st["x"].dtype
    x, w, b = st["x"].float(), st["w"].float(), st["b"].float()
    z = x @ w.t() + b
    erf = torch.erf(z * math.sqrt(0.5)) if case["act"] == "gelu" else None
    y = (0.5 * z * (1 + erf) if case["act"] == "gelu"
         else torch.where(z > 0, z, torch.zeros_like(z)) if case["act"] == "relu" else z)
    if st["r"] is not None:
        y = y + st["r"].float()
    if not case["train"]:
        return y.to(dt)
    dz = st["gy"].float()
    if case["act"] == "gelu":
        dz = dz * (0.5 * (1 + erf) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    elif case["act"] == "relu":
        dz = dz * (z > 0)
    return y.to(dt), (dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt)


def _plain_attention(st):
    """A padded batch: [W, kv heads, queries of the group's heads, keys]."""
    case, dt = st["case"], st["q"].dtype
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    grp, (rq, oq), (rk, ok) = h // hkv, st["rows_q"], st["rows_k"]
    nw, lq, lk = len(st["nq"]), rq.shape[1], rk.shape[1]
    scale = 1 / math.sqrt(d)

    def heads_first(t, rows, there, n_heads):
        t = torch.where(there[..., None, None], t.float()[rows], torch.zeros((), device=DEV))
        return t.permute(0, 2, 1, 3).reshape(nw, hkv, n_heads // hkv * rows.shape[1], d)

    q = heads_first(st["q"], rq, oq, h)
    k, v = (heads_first(st[n], rk, ok, hkv) for n in "kv")
    s = (q @ k.transpose(2, 3)).view(nw, hkv, grp, lq, lk) * scale
    seen = ok[:, None, :].expand(nw, lq, lk)
    if case["causal"]:
        i, j = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)
        ahead = torch.tensor(st["nk"], device=DEV) - torch.tensor(st["nq"], device=DEV)
        seen = seen & (j <= (i[None, :] + ahead[:, None])[..., None])
    if st["table"] is not None:
        ids = st["pad_ids"].long()
        seen = seen & (ids < case["buckets"])
        ids = torch.where(seen, ids, case["buckets"])
        table = torch.cat([st["table"].float(), torch.zeros(1, h, device=DEV)])
        s += table[ids].permute(0, 3, 1, 2).view(nw, hkv, grp, lq, lk)
    s = torch.where(seen[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(nw, hkv, grp * lq, lk)
    o = p @ v

    def rows_first(t, there, n_heads):
        t = t.view(nw, n_heads, there.shape[1], d).permute(0, 2, 1, 3)
        return t[there].to(dt)

    if not case["train"]:
        return rows_first(o, oq, h)
    g = heads_first(st["go"], rq, oq, h)
    dp = g @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    out = [rows_first(o, oq, h), rows_first(ds @ k * scale, oq, h),
           rows_first(ds.transpose(2, 3) @ q * scale, ok, hkv),
           rows_first(p.transpose(2, 3) @ g, ok, hkv)]
    if st["table"] is not None:
        # one column of ones for each bucket; a query's keys in 32 bits, the queries in 64
        one = (ids[..., None] == torch.arange(case["buckets"], device=DEV)).float()
        per_query = ds.view(nw, h, lq, lk).transpose(1, 2).contiguous() @ one
        out.append(per_query.double().sum((0, 1)).t().to(dt))
    return tuple(out)


# ----------------------------------------------------------- work and the truth
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        byte = es * (m * k + n * k + n + m * n * (2 if case["residual"] else 1))
        if case["train"]:
            byte += es * (m * n + m * k + n * k + n)
        return {"bytes": byte, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    nq, nk = _both_lengths(case)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = 0
    for a, b in zip(nq, nk):
        first = min(b, max(0, b - a + 1)) if case["causal"] else b
        pairs += (first + b) * a // 2 if case["causal"] else a * b
    byte = es * d * (2 * sum(nq) * h + 2 * sum(nk) * hkv)
    if case["train"]:
        byte += es * d * (2 * sum(nq) * h + 2 * sum(nk) * hkv)
    if case["kind"] == "bias":
        byte += sum(a * b for a, b in zip(nq, nk)) + es * case["buckets"] * h * (
            2 if case["train"] else 1)
    return {"bytes": byte, "flops": pairs * h * d * (14 if case["train"] else 4)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        x, w, b = (st[n].detach().double().requires_grad_(case["train"]) for n in "xwb")
        z = torch.einsum("mk,nk->mn", x, w) + b
        y = (torch.nn.functional.gelu(z) if case["act"] == "gelu"
             else torch.clamp(z, min=0) if case["act"] == "relu" else z)
        if st["r"] is not None:
            y = y + st["r"].double()
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), st["gy"].double()))
    names = ["q", "k", "v"] + (["table"] if st["table"] is not None else [])
    leaf = {n: st[n].detach().double() for n in names}
    grads = {n: torch.zeros_like(t) for n, t in leaf.items()}
    grp = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(leaf["q"])
    aq = ak = ap = 0
    for a, b in zip(st["nq"], st["nk"]):
        seen = torch.ones(a, b, dtype=torch.bool, device=DEV)
        if case["causal"]:
            seen = seen.tril(b - a)
        ids = None
        if "table" in leaf:
            ids = st["ids"][ap:ap + a * b].view(a, b).long()
            seen = seen & (ids < case["buckets"])
            ids = ids.clamp(max=case["buckets"] - 1)
            ap += a * b
        for head in range(case["heads"]):
            one = [leaf["q"][aq:aq + a, head], leaf["k"][ak:ak + b, head // grp],
                   leaf["v"][ak:ak + b, head // grp]]
            one += [leaf["table"][:, head]] if ids is not None else []
            one = [t.clone().requires_grad_(case["train"]) for t in one]
            s = one[0] @ one[1].t() / math.sqrt(case["dim"])
            if ids is not None:
                s = s + one[3][ids]
            s = s.masked_fill(~seen, -math.inf)
            none = ~seen.any(1, keepdim=True)
            o = torch.softmax(s.masked_fill(none, 0.0), 1).masked_fill(none, 0.0) @ one[2]
            out[aq:aq + a, head] = o.detach()
            if case["train"]:
                got = torch.autograd.grad(o, one, st["go"][aq:aq + a, head].double())
                grads["q"][aq:aq + a, head] += got[0]
                grads["k"][ak:ak + b, head // grp] += got[1]
                grads["v"][ak:ak + b, head // grp] += got[2]
                if ids is not None:
                    grads["table"][:, head] += got[3]
        aq, ak = aq + a, ak + b
    return (out, *(grads[n] for n in names)) if case["train"] else out
