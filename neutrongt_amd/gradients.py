"""The global norm of a model's gradients, and clipping by it, on the HIP kernels.

The step between a backward pass and the optimizer: a few launches for all tensors
together, no copy of their addresses to the GPU, no synchronisation with the host, so
that it can be part of a captured training step (``encoder.window_step``'s
``max_grad_norm``).  The reference's training step
(NeutronGT/core/node_level_pipeline/train_eval.py:255-300) does not clip.

Every compute call goes through libngt_attn.so; there is no PyTorch/CPU
fallback (CPU tensors raise).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .attention import _DTYPES, _stream, _workspace


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one run of memory, in whatever order."""
    want = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if s != want:
            return False
        want *= n
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return all(s == r for s, r, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _check(t: torch.Tensor, name: str, dev) -> None:
    if t.layout != torch.strided:
        raise ValueError(f"{name} must be dense, got {t.layout}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (there is no CPU path)")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the others on {dev}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} has dtype {t.dtype} (float32 or bfloat16)")
    if t.numel() and not _dense(t):
        raise ValueError(f"{name} must fill one run of memory, got shape {tuple(t.shape)} and "
                         f"strides {t.stride()}")


def _run(parameters, max_norm: float, out):
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    out = list(out) if out is not None else None
    ext = _lib.autograd_ext()
    norm = ext and ext.clip_gradients(params, out, max_norm)
    if norm is not None:
        return norm
    grads = [p.grad for p in dict.fromkeys(params) if p.grad is not None]
    if out is not None and len(out) != len(grads):
        raise ValueError(f"{len(out)} results for {len(grads)} gradients")
    if not grads:
        dev = params[0].device if params else torch.device("cuda", torch.cuda.current_device())
        return torch.zeros((), dtype=torch.float32, device=dev)
    dev = grads[0].device
    for i, g in enumerate(grads):
        _check(g, f"gradient {i}", dev)
    for i, (o, g) in enumerate(zip(out or (), grads)):
        _check(o, f"result {i}", dev)
        if o.shape != g.shape or (g.numel() and not _same_order(o, g)):
            raise ValueError(f"result {i} must have its gradient's shape and strides, got "
                             f"{tuple(o.shape)} {o.stride()}")
    written = out if out is not None else grads if max_norm >= 0 else []
    runs = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w, i)
                   for ts, w in ((grads, False), (out or [], True)) for i, t in enumerate(ts)
                   if t.numel()])
    end = (0, None, None)  # the furthest end so far, of which tensor
    for a, b, w, i in runs:
        # a result may lie in its own gradient's memory, nothing else may overlap
        if a < end[0] and max_norm >= 0 and not (
                end[2] == i and end[1] != w and out[i].data_ptr() == grads[i].data_ptr()
                and out[i].dtype == grads[i].dtype):
            raise ValueError(f"gradients or results {end[2]} and {i} overlap")
        end = max(end, (b, w, i), key=lambda e: e[0])
    table = (_lib.GradientC * len(grads))()
    for i, g in enumerate(grads):
        table[i].x, table[i].n, table[i].dtype = g.data_ptr(), g.numel(), _DTYPES[g.dtype]
        if out is not None:
            table[i].out, table[i].out_dtype = out[i].data_ptr(), _DTYPES[out[i].dtype]
    lib, nb = _lib.load(), C.c_size_t()
    _lib.check(lib.ngt_clip_workspace_bytes(table, len(grads), C.byref(nb)))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(nb.value, dev)
    with torch.cuda.device(dev):
        _lib.check(lib.ngt_clip_gradients(table, len(grads), max_norm, norm.data_ptr(),
                                          ws.data_ptr(), nb.value, _stream(dev)))
    if written:
        torch.autograd.graph.increment_version(written)
    return norm


def clip_gradients(parameters, max_norm: float, out=None) -> torch.Tensor:
    """Scales the parameters' gradients together by min(1, max_norm / norm), norm being
    the 2-norm over all of them, and returns the norm (fp32, on the GPU; nothing waits
    for it).

    parameters: a tensor or an iterable; those without a gradient are skipped, one that
    is given twice counts once.  Gradients are fp32 or bf16, on one GPU, each filling
    one run of memory.  ``out``: tensors that take the scaled gradients instead, one
    for each gradient, of its shape and strides, fp32 or bf16 (e.g. fp32 gradients of
    bf16 ones for the optimizer).  The norm is summed in fp64 in a fixed order.  Where
    the one returned is not finite (a gradient holds a NaN or an infinity, or the norm is
    above fp32's range) nothing is scaled, and where it is at most max_norm the gradients'
    memory is left alone."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return _run(parameters, max_norm, out)


def gradient_norm(parameters) -> torch.Tensor:
    """The 2-norm over all gradients of the parameters, as clip_gradients returns it;
    nothing is scaled."""
    return _run(parameters, -1.0, None)
