"""neutrongt_amd -- MI355X (gfx950) window attention for NeutronGT.

Public API
----------
CoreAttention            drop-in for NeutronGT's CoreAttention (sparse + full)
install(model)           swap a model's local_attn modules for CoreAttention
sparse_attention(...)    functional masked attention over a window edge_index
window_attention(...)    the same over a built WindowAdjacency (C++ autograd node)
dense_attention(...)     functional full-window attention
packed_attention(...)    attention over a PackedWindows batch (grouped heads, causal, bucket bias)
PackedWindows            plan of windows of different lengths back to back
linear_epilogue(...)     act(x W^T + b) + residual as one kernel, differentiable
gated_linear(...)        act(x Wg^T + bg) * (x Wu^T + bu) as one kernel, differentiable
norm_rotary(...)         RMS norm and position rotation of query and key heads, differentiable
Rotary                   the angles of such a rotation
clip_gradients(...)      gradients scaled to a largest global norm; gradient_norm(...): the norm
WindowAdjacency          device CSR/transposed CSR/work lists of one window
"""
from .attention import (CoreAttention, DenseAttentionBiasFunction, DenseAttentionFunction,
                        SparseAttentionBiasFunction, SparseAttentionFunction, dense_attention,
                        dense_attention_bias, install, sparse_attention, window_attention)
from .csr import (AdjacencyCache, WindowAdjacency, chunk_for_heads, default_cache, pack_q_adaptive,
                  small_for_heads)
from .gradients import clip_gradients, gradient_norm
from .linear import GatedLinearFunction, LinearEpilogueFunction, gated_linear, linear_epilogue
from .packed import PackedAttentionFunction, PackedWindows, PairBuckets, packed_attention
from .rotary import NormRotaryFunction, Rotary, norm_rotary

__all__ = [
    "CoreAttention",
    "install",
    "sparse_attention",
    "window_attention",
    "dense_attention",
    "SparseAttentionFunction",
    "SparseAttentionBiasFunction",
    "DenseAttentionFunction",
    "DenseAttentionBiasFunction",
    "dense_attention_bias",
    "packed_attention",
    "PackedAttentionFunction",
    "PackedWindows",
    "PairBuckets",
    "linear_epilogue",
    "LinearEpilogueFunction",
    "gated_linear",
    "GatedLinearFunction",
    "norm_rotary",
    "NormRotaryFunction",
    "Rotary",
    "clip_gradients",
    "gradient_norm",
    "WindowAdjacency",
    "AdjacencyCache",
    "chunk_for_heads",
    "pack_q_adaptive",
    "small_for_heads",
    "default_cache",
]
