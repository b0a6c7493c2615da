"""The angles of Rotary under its scalings, against the formulas computed here pair by pair,
and norm_rotary's results with them."""
import math

import pytest
import torch

from neutrongt_amd import Rotary, norm_rotary
from oracle import rotary as OR

pytestmark = pytest.mark.gpu
F32 = torch.float32


def _plain(dim, base=10000.0):
    return [base ** (-2 * i / dim) for i in range(dim // 2)]


def _base(dim, factor, base=10000.0):
    """The geometric series from 1 to its last term divided by factor."""
    last = base ** (-(dim - 2) / dim) / factor
    return [last ** (i / (dim // 2 - 1)) for i in range(dim // 2)]


def _parts(dim, factor, length, slow, fast, base=10000.0):
    f = []
    for v in _plain(dim, base):
        turns = v * length / (2 * math.pi)
        if turns >= fast:
            f.append(v)
        elif turns <= slow:
            f.append(v / factor)
        else:
            share = (turns - slow) / (fast - slow)
            f.append(v * share + v / factor * (1 - share))
    return f


CASES = [
    (dict(), 16, _plain(16), 1.0),
    (dict(base=500.0), 24, _plain(24, 500.0), 1.0),
    (dict(scaling="linear", factor=4.0), 16, [v / 4 for v in _plain(16)], 1.0),
    (dict(scaling="linear", factor=0.5, magnitude=0.7), 6, [2 * v for v in _plain(6)], 0.7),
    (dict(scaling="base", factor=8.0), 32, _base(32, 8.0), 1.0),
    (dict(scaling="base", factor=2.0, base=100.0), 4, _base(4, 2.0, 100.0), 1.0),
    (dict(scaling="base", factor=8.0), 2, [1.0], 1.0),
    (dict(scaling="parts", factor=4.0, trained_length=2048), 64, _parts(64, 4.0, 2048, 1, 32),
     0.1 * math.log(4.0) + 1),
    (dict(scaling="parts", factor=16.0, trained_length=500, slow=2.0, fast=9.0, base=300.0), 24,
     _parts(24, 16.0, 500, 2, 9, 300.0), 0.1 * math.log(16.0) + 1),
    (dict(scaling="parts", factor=4.0, trained_length=2048, magnitude=1.0), 64,
     _parts(64, 4.0, 2048, 1, 32), 1.0),
    (dict(scaling="parts", factor=0.5, trained_length=100), 8, _parts(8, 0.5, 100, 1, 32), 1.0),
    (dict(frequencies=[1.0, -0.25, 0.0, 3.5], magnitude=2.0), 8, [1.0, -0.25, 0.0, 3.5], 2.0),
]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_scalings(dev, i, layout):
    kw, dim, f, magnitude = CASES[i]
    rot = Rotary(dim, layout=layout, device=dev, **kw)
    f = torch.tensor(f, dtype=torch.float64)
    # fp64 powers: some 2^-50 of each
    assert ((rot.frequencies - f).abs() <= 1e-14 * f.abs()).all()
    assert ((rot.turns.cpu() * 2 * math.pi - f).abs() <= 1e-14 * f.abs()).all()
    assert abs(rot.magnitude - magnitude) <= 1e-15 * magnitude
    g = torch.Generator().manual_seed(i)
    x, gy = (torch.randn(40, 3, dim + 6, generator=g) for _ in range(2))
    pos = torch.randint(-3000, 3001, (40,), generator=g)
    xd = x.to(dev).requires_grad_()
    y = norm_rotary(xd, positions=pos.to(dev), rotary=rot)
    dx, = torch.autograd.grad(y, xd, gy.to(dev))
    ref = OR.bounds(x, None, pos, f, layout, magnitude, 1e-6, gy, 2.0 ** -24, 0.0)
    for got, (want, bound) in zip((y.detach(), dx), ref):
        assert ((got.double().cpu() - want).abs() <= bound).all()


def test_the_ends_of_the_scalings():
    """What the documentation says of each: "base" leaves the fastest pair alone and divides
    the slowest by factor; "parts" has both kinds, and pairs between them."""
    assert _base(32, 8.0)[0] == 1.0 and _base(32, 8.0)[-1] == pytest.approx(_plain(32)[-1] / 8)
    by = [a / b for a, b in zip(_parts(64, 4.0, 2048, 1, 32), _plain(64))]
    assert by[0] == 1.0 and by[-1] == 0.25 and any(0.25 < v < 1.0 for v in by)
    assert all(a >= b for a, b in zip(by, by[1:]))
