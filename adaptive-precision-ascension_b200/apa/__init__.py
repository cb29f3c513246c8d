"""Adaptive Precision Ascension on B200.

Drop-in for the reference package ``apa``: the same public names
(apa/__init__.py:1-15), with APALinear's casts, GEMMs and telemetry and the
manager's ladder running as sm_100a kernels from libapa_kernels.so. Beside
them ``apa.blockscale``: E4M3 tensors with one scale per 128 elements, a linear
layer on them and the root-mean-square norm in front of it.
"""
from .config import APAConfig
from .layers import APALinear, APABoundaryCast
from .manager import APAManager
from .telemetry import APAForensicLogger
from .blockscale import (APABlockLinear, APABlockTensor, APARMSNorm, block_cast, block_linear, block_matmul,
                         rms_norm)

__version__ = "0.1.0"

__all__ = [
    "APAConfig",
    "APALinear",
    "APABoundaryCast",
    "APAManager",
    "APAForensicLogger",
    "APABlockLinear",
    "APABlockTensor",
    "APARMSNorm",
    "block_cast",
    "block_linear",
    "block_matmul",
    "rms_norm",
    "__version__",
]
