"""RMSNorm wrapper (reference: aot_kernel/norm.py:9-18)."""

import torch

from . import _C  # noqa: F401  (registers torch.ops.aot_kernel.*)
from .utils import assert_contiguous, assert_same_device, assert_same_dtype

_sandwich_rmsnorm = torch.ops.aot_kernel.sandwich_rmsnorm.default


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """y = x * rsqrt(mean(x**2, -1) + eps) * weight over the last dim, fp32 math."""
    if not x.is_cuda:
        raise ValueError("cuda rmsnorm requires a CUDA tensor")
    assert_contiguous(x, weight)
    assert_same_device(x, weight)
    assert_same_dtype(x, weight)
    out = torch.empty_like(x)
    torch.ops.aot_kernel.rmsnorm_forward(out, x, weight, eps)
    return out


rms_norm = rmsnorm


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(rmsnorm(h, weight, eps), h) with h = x + residual rounded to the dtype.

    The pre-norm step of a transformer block in one pass: equal to
    ``rmsnorm(x + residual, weight, eps)`` and ``x + residual``.
    """
    if not x.is_cuda:
        raise ValueError("cuda add_rmsnorm requires a CUDA tensor")
    assert_contiguous(x, residual, weight)
    assert_same_device(x, residual, weight)
    assert_same_dtype(x, residual, weight)
    if x.shape != residual.shape:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)} vs residual {tuple(residual.shape)}")
    out = torch.empty_like(x)
    h = torch.empty_like(x)
    torch.ops.aot_kernel.add_rmsnorm_forward(out, h, x, residual, weight, eps)
    return out, h


def sandwich_rmsnorm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                     pre_weight: torch.Tensor, eps: float = 1e-6, *,
                     gate: torch.Tensor | None = None,
                     residual_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The norm after one residual block and the norm before the next, in one pass:

        h   = residual_scale * residual + gate * rmsnorm(x, post_weight, eps)
        out = rmsnorm(h, pre_weight, eps)

    Returns ``(out, h)`` as ``add_rmsnorm`` does, each rounded once from fp32 (out
    sees the unrounded h).  ``x`` is the block's output.  ``gate`` broadcasts over
    x: its last dim is H or 1, its leading dims match x's from the left and are 1
    after that - e.g. ``[H]`` (per channel), ``[B, 1, H]`` (per sequence),
    ``[B, S, 1]`` (per token) or x's own shape.  A factor on the block's branch
    can be folded into ``gate`` or ``post_weight``.  Rows of any finite values are
    normalised, whether or not their squares fit fp32.  All tensors are contiguous and of
    one dtype; anything else is a ValueError.  Forward only, like the other norms.
    """
    if not x.is_cuda:
        raise ValueError("cuda sandwich_rmsnorm requires a CUDA tensor")
    return _sandwich_rmsnorm(x, residual, post_weight, pre_weight, gate, residual_scale, eps)


def rms_rstd(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """fp32 rsqrt(mean(x**2, -1) + eps), one value per row: rms_norm's row
    statistic, for folding the normalisation into the next GEMM
    (``gemm_silu_mul(x, fold_norm_weight(w_gate_up, w), row_scale=rstd)``)."""
    if not x.is_cuda:
        raise ValueError("cuda rms_rstd requires a CUDA tensor")
    assert_contiguous(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    torch.ops.aot_kernel.rmsnorm_rstd(rstd, x, eps)
    return rstd
