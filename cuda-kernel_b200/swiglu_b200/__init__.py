"""B200-native batch-one SwiGLU decode layer (sm_100a).

Host-side mirror of shubhxho/cuda-kernel's operator surface over the C ABI of
``libswiglu_b200.so``:

* ``swiglu_out`` / ``swiglu`` / ``config_ids`` -- the torch binding
  (``src/torch_extension.cu``), same names, checks and errors;
* ``gate`` / ``project`` / ``ffn`` -- the kernel launches of
  ``decode::launch`` (``include/kernels.cuh:115-133``);
* ``mx4_*`` -- four-bit (MXFP4) matrices: rounding, reading back, products;
* ``moe`` -- the layer as a mixture of experts, 16-bit or four-bit weights;
* ``CublasBaseline`` -- the cuBLAS GemmEx + pointwise comparison path.

Importing this package does not need a GPU; calling a kernel does.
"""
from .binding import (CublasBaseline, config_ids, config_info, device_error, ffn, ffn_fused, ffn_tp, gate,
                      layer_config_ids, layer_workspace, project,
                      residual_epilogue, swiglu, swiglu_out, valid_config)
from .moe import moe, moe_out, moe_workspace
from .mx4 import (mx4_dequantize, mx4_dequantize_out, mx4_empty, mx4_matmul, mx4_matmul_out, mx4_project,
                  mx4_project_out, mx4_quantize, mx4_quantize_out)
from ._lib import build, lib

__all__ = ["swiglu_out", "swiglu", "config_ids", "config_info", "valid_config", "gate", "project", "ffn", "ffn_fused", "ffn_tp",
           "layer_config_ids", "layer_workspace",
           "residual_epilogue", "device_error", "CublasBaseline", "build", "lib",
           "mx4_quantize", "mx4_quantize_out", "mx4_dequantize", "mx4_dequantize_out", "mx4_empty",
           "mx4_project", "mx4_project_out", "mx4_matmul", "mx4_matmul_out", "moe", "moe_out", "moe_workspace"]
