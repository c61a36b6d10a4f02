"""Gated activations that keep their inputs in 8 bits for the backward pass."""
from .glu_act8 import (  # noqa: F401
    ForgeGLUAct8Function,
    ForgePackedGLUAct8Function,
    glu_act8,
    glu_act8_packed,
)
