from .kernel import rms_norm, rms_norm_int8
from .module import RMSNorm

__all__ = ["rms_norm", "rms_norm_int8", "RMSNorm"]
