"""Attention over packed sequences or a dense batch (csrc/attention*.hip)."""
from .attention import ForgeAttentionFunction, forge_attention, forge_varlen_attention

__all__ = ["ForgeAttentionFunction", "forge_attention", "forge_varlen_attention"]
