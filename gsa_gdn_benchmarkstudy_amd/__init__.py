"""MI355X-native Gated Sparse Attention (GSA) forward.

Drop-in for the GSA layer of nirmalpratheep/GSA_GDN_BenchmarkStudy
(``gsa_triton/gsa_opt.py``): the same module API, backed by hand-written gfx950
HIP kernels in ``libgsa_hip.so`` (C ABI: ``include/gsa_hip.h``).  Beside it, for the
study's other mixer: the gated delta rule (``gated_delta_rule`` with its backward pass,
``gated_delta_step`` for serving), linear attention with a decay for each head on the same
states (``linear_attention``, ``linear_attention_step``), attention in a sliding window with
first tokens that stay visible (``window_attention``, ``window_cache_write``,
``window_attention_step``) and the RMS norm around all of them (``add_rms_norm``,
``add_rms_norm_fp8``).
"""

from .gsa import (  # noqa: F401
    AdaptiveTopKSelector,
    GatedLightningIndexer,
    GatedSparseAttention,
    OutputGate,
    RotaryEmbedding,
    ValueGate,
    apply_rotary_pos_emb,
    fused_gated_indexer,
    fused_sparse_attention,
)
from .delta import gated_delta_rule, gated_delta_step  # noqa: F401
from .linear import linear_attention, linear_attention_step  # noqa: F401
from .norm import add_rms_norm, add_rms_norm_fp8  # noqa: F401
from .window import window_attention, window_attention_step, window_cache_write  # noqa: F401

__all__ = [
    "AdaptiveTopKSelector", "GatedLightningIndexer", "GatedSparseAttention", "OutputGate",
    "RotaryEmbedding", "ValueGate", "apply_rotary_pos_emb", "fused_gated_indexer",
    "fused_sparse_attention", "gated_delta_rule", "gated_delta_step", "linear_attention", "linear_attention_step",
    "add_rms_norm", "add_rms_norm_fp8", "window_attention", "window_attention_step", "window_cache_write",
]
