from triton_helpers_amd.layers.wide_mlp import Int8WideMLP, WideMLP  # noqa: F401

__all__ = ["Int8WideMLP", "WideMLP"]
