"""Gated activations kept in 8 bits for the backward pass (no reference
counterpart; beside forge.kernels.swiglu and forge.kernels.geglu)."""
from kernels.glu_act8 import ForgeGLUAct8Function, ForgePackedGLUAct8Function, glu_act8, glu_act8_packed

__all__ = ["ForgeGLUAct8Function", "ForgePackedGLUAct8Function", "glu_act8", "glu_act8_packed"]
