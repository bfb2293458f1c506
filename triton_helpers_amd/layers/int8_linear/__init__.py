from .kernel import int8_linear, quantize_rows
from .module import Int8Linear

__all__ = ["int8_linear", "quantize_rows", "Int8Linear"]
