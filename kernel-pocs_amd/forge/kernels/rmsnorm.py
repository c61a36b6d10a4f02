"""RMSNorm re-export (reference forge/forge/kernels/rmsnorm.py)."""
from kernels.rmsnorm import (
    ForgeAddRMSNormFunction,
    ForgeRMSNormFunction,
    add_rmsnorm,
    add_rmsnorm_int8,
    apply_rmsnorm,
    rmsnorm,
    rmsnorm_backward,
    rmsnorm_forward,
    torch_rmsnorm_reference,
)

__all__ = [
    "ForgeAddRMSNormFunction",
    "ForgeRMSNormFunction",
    "add_rmsnorm",
    "add_rmsnorm_int8",
    "apply_rmsnorm",
    "rmsnorm",
    "rmsnorm_backward",
    "rmsnorm_forward",
    "torch_rmsnorm_reference",
]
