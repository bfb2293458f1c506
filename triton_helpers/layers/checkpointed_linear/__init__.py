from triton_helpers_amd.layers.checkpointed_linear import CheckpointedLinear, checkpointed_linear  # noqa: F401

__all__ = ["checkpointed_linear", "CheckpointedLinear"]
