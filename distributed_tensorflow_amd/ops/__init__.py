"""Fused ops: gfx950 HIP kernels (``hip_backend``), their PyTorch fp32 oracle (``reference``), the differentiable MatMul on the
hand-written GEMM (``gemm``), and what a model over tokens trains with: table lookup (``embedding``), cross-entropy against
integer labels (``xent``), orthogonalised updates of matrices (``muon``)."""
from . import embedding, gemm, hip_backend, muon, reference, xent  # noqa: F401
from .reference import ACT_RELU, ACT_SIGMOID, act_code  # noqa: F401
