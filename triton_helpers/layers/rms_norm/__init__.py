from triton_helpers_amd.layers.rms_norm import RMSNorm, rms_norm, rms_norm_int8  # noqa: F401

__all__ = ["rms_norm", "rms_norm_int8", "RMSNorm"]
