"""Attention re-export (no reference counterpart)."""
from kernels.attention import ForgeAttentionFunction, forge_attention, forge_varlen_attention

__all__ = ["ForgeAttentionFunction", "forge_attention", "forge_varlen_attention"]
