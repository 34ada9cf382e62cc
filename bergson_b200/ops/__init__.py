"""Operators: model-side ops (``functional``), attribution kernels (``attribution``)
and the loader of the in-tree sm_100a extension (``native``)."""

from .linear import Linear, linear
from .functional import (
    causal_attention,
    composable,
    gelu,
    layer_norm,
    rms_norm,
    rotary,
    rotary_tables,
    swiglu,
    token_cross_entropy,
    token_distillation,
    use_fused,
)
from .packed import PackedSequences, packed_causal_attention, packed_rotary

__all__ = [
    "Linear",
    "PackedSequences",
    "linear",
    "causal_attention",
    "composable",
    "gelu",
    "layer_norm",
    "packed_causal_attention",
    "packed_rotary",
    "rms_norm",
    "rotary",
    "rotary_tables",
    "swiglu",
    "token_cross_entropy",
    "token_distillation",
    "use_fused",
]
