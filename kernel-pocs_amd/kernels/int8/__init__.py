"""Linear layers on frozen 8-bit weights (csrc/int8_gemm.hip)."""
from .int8 import Int8LinearFunction, Int8Rows, Int8Weight, int8_linear, quantize_int8_rows

__all__ = ["Int8LinearFunction", "Int8Rows", "Int8Weight", "int8_linear", "quantize_int8_rows"]
