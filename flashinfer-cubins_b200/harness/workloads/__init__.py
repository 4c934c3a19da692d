"""Importing this package registers the NVFP4 and INT8 workloads."""

from . import int8, nvfp4_dual_gemm, nvfp4_gemm, nvfp4_group_gemm  # noqa: F401
