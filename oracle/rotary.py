"""RMS norm and position rotation of heads, restated in float64, with gradients from
torch.autograd and, for a kernel that computes in fp32 and rounds its results, how far
each may be from these."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def pairs(dim, layout):
    """The first and second components of the rotated pairs."""
    if layout == "half":
        return torch.arange(dim // 2), torch.arange(dim // 2, dim)
    return torch.arange(0, dim, 2), torch.arange(1, dim, 2)


def rotate(u, angle, layout, magnitude=1.0):
    """u [n, H, d] with the first 2 angle.shape[1] components turned by angle [n, dim / 2]."""
    dim = 2 * angle.shape[1]
    a, b = pairs(dim, layout)
    c, s = (f(angle)[:, None] * magnitude for f in (torch.cos, torch.sin))
    cols = [u[..., i] for i in range(u.shape[-1])]
    for i, (p, q) in enumerate(zip(a.tolist(), b.tolist())):
        cols[p] = u[..., p] * c[..., i] - u[..., q] * s[..., i]
        cols[q] = u[..., p] * s[..., i] + u[..., q] * c[..., i]
    return torch.stack(cols, -1)


def forward(x, gain, positions, frequencies, layout, magnitude=1.0, eps=1e-6):
    """x [n, H, d] and gain [d] (or None) in float64; positions [n] with frequencies
    [dim / 2], or None and None."""
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain
    if positions is None:
        return x
    return rotate(x, positions.double()[:, None] * frequencies, layout, magnitude)


def bounds(x, gain, positions, frequencies, layout, magnitude, eps, gy, half, gain_half):
    """[(y, bound), (dx, bound), (dgain, bound) or None].

    u = 2^-24 is fp32's half step.  The sum of d squares and what follows leave s =
    1 / sqrt(..) within (d / 2 + 6) u of itself, h = x s and u = h gain within
    (d / 2 + 8) u.  A cosine or sine is off by 8 u (its argument, below an eighth of
    a turn, rounded; the function; the magnitude) and by what fp64 loses of the
    angle, 2^-51 of it.  Every other product and sum adds u of its terms."""
    n, H, d = x.shape
    X = x.detach().double().clone().requires_grad_()
    G = gain.detach().double().clone().requires_grad_() if gain is not None else None
    y = forward(X, G, positions, frequencies, layout, magnitude, eps)
    leaves = [X] + ([G] if G is not None else [])
    grads = torch.autograd.grad(y, leaves, gy.double())
    with torch.no_grad():
        X = X.detach()
        s = (1 / torch.sqrt((X * X).mean(-1, keepdim=True) + eps) if gain is not None
             else torch.ones(n, H, 1, dtype=torch.float64))
        h = X * s
        u = h * (G if gain is not None else 1.0)
        e_u = (d / 2 + 8) * U if gain is not None else 0.0
        mix_u, mix_g, e_t = u.abs(), gy.double().abs(), torch.zeros(n, H, d, dtype=torch.float64)
        g = gy.double()
        if positions is not None:
            angle = positions.double()[:, None] * frequencies
            a, b = pairs(2 * angle.shape[1], layout)
            g = rotate(g / 1.0, -angle, layout, magnitude)
            for m in (mix_u, mix_g):
                both = (m[..., a] + m[..., b]) * abs(magnitude)
                m[..., a] = m[..., b] = both
            e = 8 * U + angle.abs() * 2.0 ** -51
            e_t[..., a] = e_t[..., b] = e[:, None].expand(n, H, -1) + 3 * U
        e_y = mix_u * (e_u + e_t)
        out = [(y.detach(), e_y + half * (y.detach().abs() + e_y))]
        e_g = mix_g * e_t
        w = g * (G if gain is not None else 1.0)
        e_w = e_g * (G.abs() if gain is not None else 1.0) + U * w.abs()
        if gain is None:
            dx, e = w, e_g
        else:
            wh = (w * h).abs()
            mean = (w * h).mean(-1, keepdim=True)
            e_m = (e_w * h.abs() + (d / 2 + 9) * U * wh).mean(-1, keepdim=True) + (
                d + 2) * U * wh.mean(-1, keepdim=True)
            dx = grads[0]
            e = s * (e_w + h.abs() * e_m + (d / 2 + 9) * U * (h * mean).abs()
                     + 2 * U * (w.abs() + (h * mean).abs())) + (d / 2 + 8) * U * dx.abs()
        out.append((grads[0], e + half * (dx.abs() + e)))
        if gain is None:
            out.append(None)
        else:
            e = (e_g * h.abs() + (d / 2 + 9) * U * (g * h).abs()).sum((0, 1)) + (
                n * H * U * (g * h).abs().sum((0, 1)))
            out.append((grads[1], e + gain_half * (grads[1].abs() + e)))
    return out
