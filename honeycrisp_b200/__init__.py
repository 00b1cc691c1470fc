"""honeycrisp_b200: sm_100a implementation of Honeycrisp's dense matrix-product path.

Public surface:
  CUDABackend, CUDAData, DType, BackendError (+ subclasses)  - honeycrisp_b200.backend
  Tensor, matmul, batchedMatmul                               - honeycrisp_b200.linalg
  Linear (fused forward, on-device backward)                  - honeycrisp_b200.linear
  LayerNorm, FeedForward, Experts, AdamW                      - honeycrisp_b200.feedforward
  shardBatch, columnBlock, batchedMatmulSharded, matmulColumnSplit - honeycrisp_b200.sharding
The compute library is honeycrisp_b200/libhccuda.so (C ABI in include/hc_cuda.h).
"""
from .backend import (AdamWPlan, AllocationFailed, BackendError, CUDABackend, CUDAData, DeviceTimeout, DType,
                      KernelFailed, NotImplementedByBackend)
from .linalg import Tensor, batchedMatmul, matmul
from .linear import Linear
from .feedforward import AdamW, Experts, FeedForward, LayerNorm

__all__ = [
    "AdamW", "AdamWPlan", "AllocationFailed", "BackendError", "CUDABackend", "CUDAData", "DeviceTimeout", "DType", "Experts", "FeedForward",
    "KernelFailed", "LayerNorm", "Linear", "NotImplementedByBackend", "Tensor", "batchedMatmul", "matmul",
]
