from triton_helpers_amd.layers.int8_linear import Int8Linear, int8_linear, quantize_rows  # noqa: F401

__all__ = ["int8_linear", "quantize_rows", "Int8Linear"]
