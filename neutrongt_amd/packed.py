"""Attention over packed windows on the HIP kernels: several windows of different
lengths in one call, grouped heads, causal order, a learned bias per pair bucket.

``dense_attention`` runs one window; here a batch of windows (the small
graphs of a graph-level task, the partitions of a node-level one, requests that
attend to cached keys) lies back to back along the rows, without padding.
``PackedWindows`` is the plan of such a batch, built once per set of lengths and
shared by all layers and steps.

The bias is the structural encoding of the reference's ``struct_enc`` models
(an embedding of each pair's hop distance per head, built there as a dense
[1, H, N, N] ``attn_bias``: NeutronGT/models/graphormer_dist_node_level.py:
308-324): ``bias_table`` [n_buckets, H] is that embedding's weight and
``PairBuckets`` the pairs' ids, one byte a pair for all heads.  Nothing of size
H x N x N exists; the table gets its gradient.

Every compute call goes through libngt_attn.so; there is no PyTorch/CPU
fallback (CPU tensors raise).
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _dtype_code, _prep, _stream, _workspace


def _lengths(x, name: str) -> torch.Tensor:
    t = torch.as_tensor(x if len(x) else torch.empty(0, dtype=torch.int32), device="cpu")
    if t.dim() != 1 or t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise ValueError(f"{name} must be a 1-D sequence of integers, got {tuple(t.shape)} {t.dtype}")
    if t.numel() and (int(t.min()) < 0 or int(t.max()) > 1 << 28):
        raise ValueError(f"{name} must lie in [0, 2^28]")
    return t.to(torch.int32).contiguous()


class PackedWindows:
    """Plan of a batch of windows: window w owns q_lengths[w] consecutive query
    rows and k_lengths[w] consecutive key rows (default: the same).  Lengths may
    be zero.  ``causal``: query i of a window sees its keys
    j <= i + (k_length - q_length).  Lengths are host integers; the plan is
    computed on the host and copied to ``device`` on its current stream."""

    def __init__(self, q_lengths, k_lengths=None, causal: bool = False, device="cuda"):
        lib = _lib.load()
        ql = _lengths(q_lengths, "q_lengths")
        kl = ql if k_lengths is None else _lengths(k_lengths, "k_lengths")
        if ql.numel() != kl.numel():
            raise ValueError(f"{ql.numel()} query lengths but {kl.numel()} key lengths")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("device must be a GPU (the attention core has no CPU path)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        n = ql.numel()
        nb = C.c_size_t()
        _lib.check(lib.ngt_packed_plan_bytes(n, ql.data_ptr(), kl.data_ptr(), C.byref(nb)))
        host = torch.empty(nb.value, dtype=torch.uint8)
        self.mem = torch.empty(nb.value, dtype=torch.uint8, device=dev)
        self.struct = _lib.PackedWindowsC()
        _lib.check(lib.ngt_packed_plan(n, ql.data_ptr(), kl.data_ptr(), int(bool(causal)),
                                       host.data_ptr(), nb.value, self.mem.data_ptr(),
                                       C.byref(self.struct)))
        self.mem.copy_(host)
        self.device = dev
        self.stream = _stream(dev)  # the memory's own
        # the struct's bytes, for the C++ node
        self.struct_bytes = torch.frombuffer(bytearray(self.struct), dtype=torch.uint8)
        self.q_lengths, self.k_lengths = ql.tolist(), kl.tolist()
        self.causal = bool(causal)

    @property
    def n_windows(self) -> int:
        return self.struct.n_windows

    @property
    def n_q(self) -> int:
        return self.struct.n_q

    @property
    def n_k(self) -> int:
        return self.struct.n_k

    def ptr(self):
        return C.byref(self.struct)

    def on_current_stream(self) -> None:
        """Keeps the plan's memory from being reused before the work that the
        current stream is about to get has run."""
        if _stream(self.device) != self.stream:
            self.mem.record_stream(torch.cuda.current_stream(self.device))

    def workspace_bytes(self, dtype: int, heads: int, kv_heads: int, dim: int, n_buckets: int = 0):
        f, b = C.c_size_t(), C.c_size_t()
        _lib.check(_lib.load().ngt_packed_workspace_bytes(dtype, self.ptr(), heads, kv_heads, dim,
                                                          n_buckets, C.byref(f), C.byref(b)))
        return f.value, b.value

    def pack_buckets(self, ids) -> "PairBuckets":
        """The pairs' bucket ids in the kernels' layouts (by queries and by
        keys).  ``ids``: a 1-D integer tensor, the windows' [queries, keys]
        matrices back to back, or a list of those matrices.  A pair whose id is
        negative or not below the table's n_buckets (at most 255, so 255 always)
        is not attended."""
        if isinstance(ids, (list, tuple)):
            if len(ids) != self.n_windows or any(
                    tuple(t.shape) != s for t, s in zip(ids, zip(self.q_lengths, self.k_lengths))):
                raise ValueError("ids must hold one [queries, keys] matrix per window")
            ids = torch.cat([t.reshape(-1) for t in ids]) if ids else torch.empty(
                0, dtype=torch.uint8, device=self.device)
        if ids.device != self.device:
            raise ValueError(f"ids are on {ids.device}, the windows on {self.device}")
        if ids.dim() != 1 or ids.numel() != self.struct.n_pairs:
            raise ValueError(f"ids must be 1-D with {self.struct.n_pairs} elements, "
                             f"got {tuple(ids.shape)}")
        if ids.dtype in (torch.int8, torch.int16):
            ids = ids.to(torch.int32)
        if ids.dtype not in (torch.uint8, torch.int32, torch.int64):
            raise TypeError(f"ids must be integers, got {ids.dtype}")
        return PairBuckets(self, ids.contiguous())


class PairBuckets:
    """Bucket ids of a batch's pairs, laid out by PackedWindows.pack_buckets."""

    def __init__(self, windows: PackedWindows, ids: torch.Tensor):
        s, dev = windows.struct, windows.device
        self.windows = windows
        self.stream = _stream(dev)  # the memory's own
        windows.on_current_stream()
        self.by_query = torch.empty(max(s.bucket_bytes_q, 1), dtype=torch.uint8, device=dev)
        self.by_key = torch.empty(max(s.bucket_bytes_k, 1), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _lib.check(_lib.load().ngt_packed_buckets(
                windows.ptr(), ids.data_ptr(), ids.element_size(), self.by_query.data_ptr(),
                self.by_key.data_ptr(), self.stream))

    def on_current_stream(self) -> None:
        """As PackedWindows.on_current_stream, of the ids."""
        if _stream(self.windows.device) != self.stream:
            for t in (self.by_query, self.by_key):
                t.record_stream(torch.cuda.current_stream(self.windows.device))


def _call_dtype(q: torch.Tensor, table: torch.Tensor | None) -> int:
    """The C entries' dtype: the rows', and whether the table is fp32."""
    f32 = table is not None and table.dtype == torch.float32
    return _dtype_code(q) | (_lib.NGT_TABLE_F32 if f32 else 0)


class PackedAttentionFunction(torch.autograd.Function):
    """out [n_q, H, d] of q [n_q, H, d], k/v [n_k, H_kv, d] over a
    PackedWindows (ngt_packed_fwd / ngt_packed_bwd); ``table`` [n_buckets, H]
    and ``buckets`` (a PairBuckets) or None and None.  The backward uses the
    forward's output in fp32 and each row's softmax statistic."""

    @staticmethod
    def forward(ctx, q, k, v, table, windows, buckets, scale, want_grad):
        n_q, H, d = q.shape
        h_kv, dev, dt = k.shape[1], q.device, _call_dtype(q, table)
        out = torch.empty(n_q, H, d, dtype=q.dtype, device=dev)
        out32 = lse = None
        if want_grad:
            # fp32: out itself
            out32 = (out if q.dtype == torch.float32
                     else torch.empty(n_q, H, d, dtype=torch.float32, device=dev))
            lse = torch.empty(H if table is None else 2 * H, n_q, dtype=torch.float32, device=dev)
        n_buckets = table.shape[0] if table is not None else 0
        fwd_bytes, _ = windows.workspace_bytes(dt, H, h_kv, d)
        ws = _workspace(fwd_bytes, dev) if fwd_bytes else None
        with torch.cuda.device(dev):
            _lib.check(_lib.load().ngt_packed_fwd(
                dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0),
                v.stride(0), windows.ptr(), H, h_kv, d, scale,
                table.data_ptr() if table is not None else None, n_buckets,
                buckets.by_query.data_ptr() if table is not None else None, out.data_ptr(),
                out32.data_ptr() if out32 is not None and out32 is not out else None,
                lse.data_ptr() if lse is not None else None,
                ws.data_ptr() if ws is not None else None, fwd_bytes, _stream(dev)))
        if want_grad:
            ctx.save_for_backward(q, k, v, table, out32, lse)
            ctx.windows, ctx.buckets, ctx.scale = windows, buckets, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out):
        q, k, v, table, out32, lse = ctx.saved_tensors
        n_q, H, d = q.shape
        h_kv, dev, dt = k.shape[1], q.device, _call_dtype(q, table)
        windows, buckets = ctx.windows, ctx.buckets
        g = _prep(g_out.to(q.dtype), "grad_out")
        gq = torch.empty(n_q, H, d, dtype=q.dtype, device=dev)
        gk = torch.empty(k.shape, dtype=q.dtype, device=dev)
        gv = torch.empty(v.shape, dtype=q.dtype, device=dev)
        want_table = table is not None and ctx.needs_input_grad[3]
        gt = torch.empty_like(table) if want_table else None
        n_buckets = table.shape[0] if table is not None else 0
        _, bwd_bytes = windows.workspace_bytes(dt, H, h_kv, d, n_buckets if want_table else 0)
        ws = _workspace(bwd_bytes, dev)
        with torch.cuda.device(dev):
            _lib.check(_lib.load().ngt_packed_bwd(
                dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0),
                v.stride(0), out32.data_ptr(), g.data_ptr(), lse.data_ptr(), windows.ptr(), H,
                h_kv, d, ctx.scale, table.data_ptr() if table is not None else None, n_buckets,
                buckets.by_query.data_ptr() if table is not None else None,
                buckets.by_key.data_ptr() if table is not None else None, gq.data_ptr(),
                gk.data_ptr(), gv.data_ptr(), gt.data_ptr() if gt is not None else None,
                ws.data_ptr(), bwd_bytes, _stream(dev)))
        return gq, gk, gv, gt, None, None, None, None


def _rows(t: torch.Tensor, name: str, n: int, dim: int) -> torch.Tensor:
    """t as [n, heads, dim] rows that the kernels can read: heads side by side,
    rows 16-byte aligned (e.g. a view of a joint [n, 3, H, d] projection), else a copy."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (the attention core has no CPU path)")
    if t.dim() != 3 or t.shape[0] != n or t.shape[2] != dim:
        raise ValueError(f"{name} must be [{n}, heads, {dim}], got {tuple(t.shape)}")
    es = t.element_size()
    if n and (t.stride(2) != 1 or t.stride(1) != dim or t.stride(0) < t.shape[1] * dim
              or t.stride(0) * es % 16 or t.stride(0) * es >= 1 << 23 or t.data_ptr() % 16):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def packed_attention(q, k, v, windows: PackedWindows, scale: float | None = None, bias_table=None,
                     buckets: PairBuckets | None = None):
    """Attention of every window's queries over its own keys:
    out = softmax(scale q k^T + bias) v per window and head, [n_q, H, d].

    q [n_q, H, d], k and v [n_k, H_kv, d] in fp32 or bf16, the rows of all
    windows back to back; H a multiple of H_kv (query head h reads key head
    h // (H // H_kv)); d a multiple of 8 up to 128.  ``scale`` (default
    1/sqrt(d); dense_attention's default is the reference's sqrt(d)) multiplies
    the products and lies in [2^-100, 2^100].  ``bias_table`` [n_buckets <= 255,
    H] of q's dtype or fp32 (an fp32 parameter beside bf16 rows goes in
    unrounded, its gradient is fp32) with ``buckets`` (windows.pack_buckets):
    adds table[id, h] to a pair's score, and leaves pairs out whose id is not in
    the table.  A query that sees no key gives zeros.  Differentiable once, in
    q, k, v and bias_table; deterministic."""
    if not isinstance(windows, PackedWindows):
        raise TypeError("windows must be a PackedWindows")
    if buckets is not None and (not isinstance(buckets, PairBuckets)
                                or buckets.windows is not windows):
        raise ValueError("buckets must come from these windows' pack_buckets")
    by = (buckets.by_query, buckets.by_key) if buckets is not None else (None, None)
    if q.is_cuda and q.dim() == 3:
        windows.on_current_stream()
        if buckets is not None:
            buckets.on_current_stream()
        ext = _lib.node_ext()
        out = ext and ext.packed_attention(
            q, k, v, bias_table, windows.struct_bytes, windows.mem, *by,
            1.0 / math.sqrt(max(q.shape[2], 1)) if scale is None else float(scale))
        if out is not None:
            return out
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [rows, heads, d], got {tuple(q.shape)} {tuple(k.shape)}")
    H, d = q.shape[1:]
    q = _rows(q, "q", windows.n_q, d)
    k = _rows(k, "k", windows.n_k, d)
    v = _rows(v, "v", windows.n_k, d)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k, v must share a dtype")
    _dtype_code(q)
    if k.shape != v.shape:
        raise ValueError(f"shape mismatch k {tuple(k.shape)} v {tuple(v.shape)}")
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"head_dim {d} is not a multiple of 8 up to 128")
    if k.shape[1] < 1 or H < 1 or H % k.shape[1]:
        raise ValueError(f"{H} query heads are not a multiple of {k.shape[1]} key heads")
    if any(t.device != windows.device for t in (q, k, v)):
        raise ValueError(f"q, k, v must be on the windows' device {windows.device}")
    if (bias_table is None) != (buckets is None):
        raise ValueError("bias_table and buckets go together")
    if bias_table is not None:
        if (bias_table.dim() != 2 or bias_table.shape[1] != H
                or not 1 <= bias_table.shape[0] <= 255
                or bias_table.dtype not in (q.dtype, torch.float32)
                or bias_table.device != q.device):
            raise ValueError(f"bias_table must be [1..255, {H}] {q.dtype} or fp32 on {q.device}, got "
                             f"{tuple(bias_table.shape)} {bias_table.dtype} on {bias_table.device}")
        bias_table = bias_table.contiguous()
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError(f"scale must lie in [2^-100, 2^100], got {scale}")
    want_grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, bias_table))
    return PackedAttentionFunction.apply(q, k, v, bias_table, windows, buckets, scale, want_grad)
