"""Attention over packed windows, restated in float64: per window and head,
softmax_j(scale q_i.k_j + table[id_ij]) v over the pairs that are seen, zero rows
where none is.  Gradients through torch.autograd, and, for a kernel that rounds,
how far each result may be from this one."""
from __future__ import annotations

import math

import torch


def windows(q_len, k_len):
    """(first query, queries, first key, keys, first pair) of each window."""
    aq = ak = ap = 0
    for a, b in zip(q_len, k_len):
        yield aq, a, ak, b, ap
        aq, ak, ap = aq + a, ak + b, ap + a * b


def seen_pairs(a, b, causal, ids=None, n_buckets=0):
    seen = torch.ones(a, b, dtype=torch.bool)
    if causal:
        seen = seen.tril(b - a)
    if ids is not None:
        seen = seen & (ids >= 0) & (ids < n_buckets)
    return seen


def _weights(s, seen):
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -math.inf)
    none = top == -math.inf
    e = torch.exp(s - torch.where(none, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def attention(q, k, v, q_len, k_len, causal=False, scale=None, table=None, ids=None):
    """out [n_q, H, d] of float64 q [n_q, H, d], k/v [n_k, H_kv, d] on the CPU;
    table [n_buckets, H] and ids (1-D, the windows' matrices back to back) or None."""
    H, d = q.shape[1:]
    grp = H // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    rows = []
    for aq, a, ak, b, ap in windows(q_len, k_len):
        i = ids[ap:ap + a * b].view(a, b).long() if ids is not None else None
        seen = seen_pairs(a, b, causal, i, table.shape[0] if table is not None else 0)
        kh = k[ak:ak + b].repeat_interleave(grp, 1).transpose(0, 1)
        vh = v[ak:ak + b].repeat_interleave(grp, 1).transpose(0, 1)
        s = q[aq:aq + a].transpose(0, 1) @ kh.transpose(1, 2) * scale
        if table is not None:
            s = s + table[torch.where(seen, i, 0)].permute(2, 0, 1)
        rows.append((_weights(s, seen) @ vh).transpose(0, 1))
    return torch.cat(rows) if rows else q.new_zeros(q.shape)


def fwd_bwd(q, k, v, go, q_len, k_len, causal=False, scale=None, table=None, ids=None):
    """[out, dq, dk, dv(, dtable)] in float64."""
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    if table is not None:
        leaves.append(table.double().requires_grad_())
    out = attention(*leaves[:3], q_len, k_len, causal, scale,
                    leaves[3] if table is not None else None, ids)
    if not out.requires_grad:
        return [out] + [torch.zeros_like(t) for t in leaves]
    grads = torch.autograd.grad(out, leaves, go.double(), allow_unused=True)
    return [out.detach()] + [torch.zeros_like(t) if g is None else g
                             for g, t in zip(grads, leaves)]


def bounds(q, k, v, go, q_len, k_len, half_step, causal=False, scale=None, table=None, ids=None):
    """Elementwise bounds on the error of [out, dq, dk, dv(, dtable)] for a kernel
    that adds in fp32 and rounds, to a type whose rounding is off by at most
    ``half_step`` of the value, the weights p, the score gradients dS and the results
    (half_step 2^-24 for fp32, which rounds nothing further).

    u = 2^-24 is fp32's half step.  A score of d products, its scaling and its
    bias is off by at most e_s = (d + 4) u (scale sum|q||k| + |bias|); an fp32
    exponential of it by e_s + 4u relative to p, the row's sum of n such terms
    by as much and n u, so that p is off by e_p = 2 e_s + (n + 12) u, plus
    half_step where it is rounded for the product.  Every other sum of n terms
    adds n u of its terms' absolute values.  D = g.out carries out's error."""
    u = 2.0 ** -24
    H, d = q.shape[1:]
    hkv = k.shape[1]
    grp = H // hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    q, k, v, go = (t.double() for t in (q, k, v, go))
    half = half_step if half_step > u else 0.0
    b_out, b_q, b_k, b_v = (torch.zeros(t.shape, dtype=torch.float64) for t in (q, q, k, k))
    b_t = torch.zeros(table.shape, dtype=torch.float64) if table is not None else None
    for aq, a, ak, b, ap in windows(q_len, k_len):
        if a == 0 or b == 0:
            continue
        i = ids[ap:ap + a * b].view(a, b).long() if ids is not None else None
        seen = seen_pairs(a, b, causal, i, table.shape[0] if table is not None else 0)
        for h in range(H):
            c = h // grp
            Q, K, V, G = q[aq:aq + a, h], k[ak:ak + b, c], v[ak:ak + b, c], go[aq:aq + a, h]
            s, mag = Q @ K.t() * scale, Q.abs() @ K.abs().t() * scale
            if table is not None:
                bias = table.double()[torch.where(seen, i, 0), h]
                s = s + bias
                mag = mag + torch.where(bias.abs() < 1e30, bias.abs(), torch.zeros_like(bias))
            p = _weights(s, seen)
            # the largest score error among a row's keys that weigh anything
            e_s = ((d + 4) * u * torch.where(p > 0, mag, 0.0)).amax(1, keepdim=True)
            e_p = 2 * e_s + (b + 12) * u
            o, absum = p @ V, p @ V.abs()
            err_o = (e_p + half + b * u) * absum
            dp = G @ V.t()
            D = (G * o).sum(1, keepdim=True)
            err_D = (G.abs() * err_o).sum(1, keepdim=True) + d * u * (G * o).abs().sum(1, keepdim=True)
            ds = p * (dp - D)
            err_ds = p * (err_D + (d + 2) * u * (G.abs() @ V.abs().t())) + (e_p + 4 * u) * ds.abs()
            r_ds = err_ds + half * (ds.abs() + err_ds)
            b_out[aq:aq + a, h] = err_o
            b_q[aq:aq + a, h] = scale * ((r_ds + (b + 2) * u * ds.abs()) @ K.abs())
            n = a * grp
            b_k[ak:ak + b, c] += scale * ((r_ds + (n + 2) * u * ds.abs()).t() @ Q.abs())
            b_v[ak:ak + b, c] += ((e_p + half + n * u) * p).t() @ G.abs()
            if table is not None:
                flat = torch.where(seen, i, 0).flatten()
                # a bucket's sum: a lane's pairs, 64 lanes, the blocks: far fewer than
                # 4096 additions in a row at these sizes
                e = torch.where(seen, err_ds + 4096 * u * ds.abs(), 0.0).flatten()
                b_t[:, h].index_add_(0, flat, e)
    ref = fwd_bwd(q, k, v, go, q_len, k_len, causal, scale, table, ids)
    out = [x + half_step * (r.abs() + x) for x, r in zip([b_out, b_q, b_k, b_v], ref)]
    if table is not None:
        out.append(b_t + half_step * (ref[4].abs() + b_t))
    return ref, out
