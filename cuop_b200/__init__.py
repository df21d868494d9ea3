"""cuop_b200 — B200-native (sm_100a) dense BLAS hot path of cuOP.

The compute lives in libcuopx.so (hand-written CUDA for sm_100a behind the C
ABI in include/cuopx.h); this package is the Python host side over that ABI.
"""
from ._native import CuopError, lib, lib_path  # noqa: F401
from .int8 import int8_gated_linear, int8_linear, quantize_int8  # noqa: F401
from .layers import (  # noqa: F401
    dropout, dropout_backward, gated_linear, gated_linear_backward, layer_norm, layer_norm_backward, linear,
    linear_backward,
)
from .muon import muon_step, orthogonalize  # noqa: F401
from .ops import (  # noqa: F401
    asum, axpy, batched_gemm, batched_gemm_host, clear_device_error, copy, device_error, dot, gather_column_blocks,
    gemm, gemv, iamax, iamin, last_kernel, launch_count, nrm2, rot, scal, swap,
)

__version__ = "0.1.0"
