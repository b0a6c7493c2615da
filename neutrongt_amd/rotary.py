"""RMS norm and position rotation of query and key heads on the HIP kernels.

What a transformer block does to its queries and keys between their projections
and ``packed_attention``: each head divided by its root mean square and multiplied
by a learned gain, and its first components turned by angles that grow with the
row's position, so that a score depends on the distance of query and key.  One pass
for both, forward and backward; either of the two alone as well.  The reference's
attention (NeutronGT/models/graphormer_dist_node_level.py:128-173) has neither.

Every compute call goes through libngt_attn.so; there is no PyTorch/CPU
fallback (CPU tensors raise).
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _dtype_code, _stream, _workspace

LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "base", "parts")


class Rotary:
    """The angles of a rotation, made once for a model.

    ``dim`` components at the start of each head (even; the rest is left as it
    is) are turned in dim / 2 pairs: pair i by position * f_i radians, f_i =
    base^(-2 i / dim).  ``layout`` "half": pair i is (i, i + dim / 2);
    "interleaved": (2 i, 2 i + 1).  ``frequencies`` (dim / 2 numbers) replaces
    the f_i, ``magnitude`` (default 1) multiplies the turned components.

    ``scaling`` stretches the angles for contexts ``factor`` times as long as
    those trained on: "linear" divides all f_i by factor; "base" raises the base
    by factor^(dim / (dim - 2)), which leaves the fastest pair alone and divides
    the slowest by factor; "parts" divides those pairs that turn less than
    ``slow`` times over ``trained_length`` positions, leaves those alone that turn
    more than ``fast`` times, goes from one to the other linearly in the turns, and
    has the magnitude 0.1 ln(factor) + 1 unless one is given."""

    def __init__(self, dim: int, base: float = 10000.0, layout: str = "half",
                 scaling: str | None = None, factor: float = 1.0,
                 trained_length: int | None = None, slow: float = 1.0, fast: float = 32.0,
                 frequencies=None, magnitude: float | None = None, device="cuda"):
        dim = int(dim)
        if dim < 0 or dim % 2:
            raise ValueError(f"dim must be even and not negative, got {dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
        base, factor = float(base), float(factor)
        if not (0 < base < math.inf and 0 < factor < math.inf):
            raise ValueError(f"base and factor must be positive, got {base} and {factor}")
        half = torch.arange(0, dim, 2, dtype=torch.float64) / max(dim, 1)
        if frequencies is not None:
            f = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").flatten().clone()
            if f.numel() != dim // 2 or not bool(torch.isfinite(f).all()):
                raise ValueError(f"frequencies must be {dim // 2} finite numbers")
        else:
            if scaling == "base" and dim > 2:
                base *= factor ** (dim / (dim - 2))
            f = base ** -half
        if scaling == "linear":
            f = f / factor
        elif scaling == "parts":
            if trained_length is None or trained_length < 1 or not slow < fast:
                raise ValueError("scaling 'parts' needs trained_length >= 1 and slow < fast")
            turns = f.abs() * trained_length / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
            f = f * keep + f / factor * (1 - keep)
            if magnitude is None:
                magnitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        magnitude = 1.0 if magnitude is None else float(magnitude)
        if not math.isfinite(magnitude):
            raise ValueError(f"magnitude must be finite, got {magnitude}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("device must be a GPU (the rotation has no CPU path)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.dim, self.layout, self.magnitude, self.device = dim, layout, magnitude, dev
        self.frequencies = f
        # whole turns per position: a far position's turns are cut off exactly
        self.turns = (f / (2 * math.pi)).to(dev)
        self.stream = _stream(dev)  # the memory's own

    def on_current_stream(self) -> None:
        """Keeps the angles' memory from being reused before the work that the
        current stream is about to get has run."""
        if _stream(self.device) != self.stream:
            self.turns.record_stream(torch.cuda.current_stream(self.device))


def _head_rows(x, gain, y=None, dy=None, dgain=None):
    """The ngt_head_rows of x [n, heads, d] (backward: None without a gain) and, backward, its
    result's gradient."""
    r = _lib.HeadRowsC()
    if x is not None:
        r.x, r.x_row, r.x_head = x.data_ptr(), x.stride(0), x.stride(1)
    r.n_heads = (x if x is not None else dy).shape[1]
    if gain is not None:
        r.gain, r.gain_dtype = gain.data_ptr(), _dtype_code(gain)
    if y is not None:
        r.y = y.data_ptr()
    if dy is not None:
        r.dy, r.dy_row, r.dy_head = dy.data_ptr(), dy.stride(0), dy.stride(1)
    if dgain is not None:
        r.dgain = dgain.data_ptr()
    return r


def _rotation(rotary, positions):
    if rotary is None:
        return None
    return _lib.RotationC(positions.data_ptr(), rotary.turns.data_ptr(), positions.element_size(),
                          rotary.dim, int(rotary.layout == "interleaved"), rotary.magnitude)


def _by(struct):
    return C.byref(struct) if struct is not None else None


def _rows(t):
    """t [n, heads, d] as the kernels read it: any strides but the last's."""
    if t.numel() and (t.stride(2) != 1 or min(t.stride()) < 0):
        t = t.contiguous()
    return t


class NormRotaryFunction(torch.autograd.Function):
    """(q', k') of q [n, H, d] and k [n, H_kv, d] or None (ngt_norm_rotary_fwd /
    ngt_norm_rotary_bwd); the backward reads the normed inputs again and keeps
    nothing else."""

    @staticmethod
    def forward(ctx, q, k, q_gain, k_gain, positions, rotary, eps):
        dev = q.device
        yq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        yk = torch.empty(k.shape, dtype=k.dtype, device=dev) if k is not None else None
        with torch.cuda.device(dev):
            _lib.check(_lib.load().ngt_norm_rotary_fwd(
                _dtype_code(q), _by(_head_rows(q, q_gain, yq)),
                _by(_head_rows(k, k_gain, yk) if k is not None else None), q.shape[0], q.shape[2],
                _by(_rotation(rotary, positions)), eps, _stream(dev)))
        # (without a gain the backward does not need the input)
        ctx.save_for_backward(q if q_gain is not None else None, k if k_gain is not None else None,
                              q_gain, k_gain, positions)
        ctx.rotary, ctx.eps = rotary, eps
        return (yq, yk) if k is not None else yq

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk=None):
        q, k, q_gain, k_gain, positions = ctx.saved_tensors
        dev, want = gq.device, ctx.needs_input_grad
        new = lambda t, wanted: torch.empty(t.shape, dtype=t.dtype, device=dev) if (
            t is not None and wanted) else None
        dq, dk, dgq, dgk = (new(t, w) for t, w in zip((gq, gk, q_gain, k_gain), want))
        gq = _rows(gq)
        gk = _rows(gk) if gk is not None else None
        n, _, d = gq.shape
        nb = C.c_size_t()
        _lib.check(_lib.load().ngt_norm_rotary_bwd_workspace_bytes(n, d, C.byref(nb)))
        ws = _workspace(nb.value, dev) if dgq is not None or dgk is not None else None
        with torch.cuda.device(dev):
            _lib.check(_lib.load().ngt_norm_rotary_bwd(
                _dtype_code(gq), _by(_head_rows(q, q_gain, dq, gq, dgq)),
                _by(_head_rows(k, k_gain, dk, gk, dgk) if gk is not None else None), n, d,
                _by(_rotation(ctx.rotary, positions)), ctx.eps,
                ws.data_ptr() if ws is not None else None, nb.value if ws is not None else 0,
                _stream(dev)))
        return dq, dk, dgq, dgk, None, None, None


def norm_rotary(q, k=None, positions=None, rotary: Rotary | None = None, q_gain=None, k_gain=None,
                eps: float = 1e-6):
    """Queries and keys as attention takes them: (q', k'), or q' alone without k.

    q [..., H, d] and k [..., H_kv, d] in fp32 or bf16, the same rows; d even, at
    most 256.  With a gain ([d], of q's dtype or fp32) each head x becomes
    x / sqrt(mean(x^2) + eps) * gain; with ``rotary`` its first rotary.dim
    components are then turned by the row's position (``positions``: int32 or int64,
    the rows' shape, any sign; angles are reduced in fp64, exact to fp32 for
    positions up to 2^28).  fp32 inside, rounded once.  q and k may be views of a
    joint projection; the results are contiguous.  Differentiable once, in q, k and
    the gains (sums in a fixed order); deterministic."""
    if rotary is not None and not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    if (rotary is None) != (positions is None):
        raise ValueError("rotary and positions go together")
    if k is None and k_gain is not None:
        raise ValueError("k_gain without k")
    eps = float(eps)
    if q.is_cuda:
        if rotary is not None and rotary.device == q.device:
            rotary.on_current_stream()
        ext = _lib.node_ext()
        out = ext and ext.norm_rotary(
            q, k, q_gain, k_gain, positions, rotary.turns if rotary is not None else None,
            rotary.layout == "interleaved" if rotary is not None else False,
            rotary.magnitude if rotary is not None else 1.0, eps)
        if out is not None:
            return (out[0], out[1]) if k is not None else out[0]
    ts = [t for t in (q, k) if t is not None]
    for name, t in zip(("q", "k"), ts):
        if not t.is_cuda:
            raise ValueError(f"{name} must be a GPU tensor (there is no CPU path)")
        if t.dim() < 2 or t.shape[-2] < 1:
            raise ValueError(f"{name} must be [..., heads, d], got {tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError("q and k must share dtype and device")
    _dtype_code(q)
    lead, d = q.shape[:-2], q.shape[-1]
    if k is not None and (k.shape[:-2] != lead or k.shape[-1] != d):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must have the same rows and "
                         "head size")
    if d % 2 or not 2 <= d <= 256:
        raise ValueError(f"head_dim {d} is not even or not within 2 .. 256")
    for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
        if g is not None and (tuple(g.shape) != (d,) or g.device != q.device
                              or g.dtype not in (q.dtype, torch.float32)):
            raise ValueError(f"{name} must be [{d}] {q.dtype} or fp32 on {q.device}, got "
                             f"{tuple(g.shape)} {g.dtype} on {g.device}")
    if rotary is not None:
        if rotary.dim > d:
            raise ValueError(f"rotary turns {rotary.dim} components, the heads have {d}")
        if rotary.device != q.device or positions.device != q.device:
            raise ValueError(f"rotary and positions must be on q's device {q.device}")
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape != lead:
            raise ValueError(f"positions must be {tuple(lead)} int32 or int64, got "
                             f"{tuple(positions.shape)} {positions.dtype}")
        positions = positions.reshape(-1).contiguous()
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    q3, k3 = (_rows(t.reshape(-1, *t.shape[-2:])) if t is not None else None for t in (q, k))
    gains = [g.contiguous() if g is not None else None for g in (q_gain, k_gain)]
    out = NormRotaryFunction.apply(q3, k3, *gains, positions, rotary, eps)
    if k is None:
        return out.view(q.shape)
    return out[0].view(q.shape), out[1].view(k.shape)
