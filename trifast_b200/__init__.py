"""B200-native triangle self-attention: a drop-in for ``trifast.triangle_attention``, and the
operators around it in a pair stack's blocks."""

from .block import dropout_add, gated_feed_forward, layer_norm  # noqa: F401
from .torch import triangle_attention, triangle_attention_ending_node  # noqa: F401

__all__ = ["triangle_attention", "triangle_attention_ending_node", "layer_norm", "gated_feed_forward",
           "dropout_add"]
