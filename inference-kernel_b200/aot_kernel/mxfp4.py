"""Microscaled 4-bit floating point (OCP MX, MXFP4): quantisation, reading back
and the product of two quantised matrices.

A row's blocks of 32 consecutive elements share a power-of-two scale; an element
is e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives).  A quantised [rows, cols]
matrix is a pair of uint8 tensors:

* codes [rows, cols / 2], the even column in the low nibble;
* scales [ceil(rows / 128), ceil(cols / 128), 512], bytes that stand for
  2^(byte - 127) (255: NaN), in the order in which the tensor cores take them
  (``mxfp4_tile_scales`` lays out row-major scales, e.g. a checkpoint's).

The reference has no 4-bit path; its 8-bit product takes operands that the caller
has quantised (jit_kernel/gemm.py:199-248).
"""

import torch

from . import _C  # noqa: F401  (registers torch.ops.aot_kernel.*)

BLOCK = 32
# The operators check their arguments and allocate (ValueError; RuntimeError for
# tensors that are not on a CUDA device).
_quantize = torch.ops.aot_kernel.mxfp4_quantize.default
_dequantize = torch.ops.aot_kernel.mxfp4_dequantize.default
_gemm = torch.ops.aot_kernel.mxfp4_gemm.default
_gemm_out = torch.ops.aot_kernel.mxfp4_gemm_out.default


def _tiles(rows: int, cols: int) -> tuple[int, int, int]:
    return ((rows + 127) // 128, (cols + 127) // 128, 512)


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [rows, cols], cols a multiple of 32; fp32, fp16 or bf16,
    contiguous or a 2-D view with contiguous rows.

    The scale of a block is 2^(floor(log2 max|x|) - 2), clamped to [2^-127, 2^127];
    x / scale is rounded to the nearest element, ties to the even code, and
    magnitudes above 6 become 6.  A block that holds a NaN or an infinity reads
    back as NaN.
    """
    return _quantize(x)


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, cols] that codes and scales stand for, rounded once to dtype."""
    return _dequantize(codes, scales, dtype)


def mxfp4_gemm(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor,
               out_dtype: torch.dtype = torch.bfloat16, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """C [M, N] = A B^T for quantised A [M, K] and B [N, K] (a weight as [out features,
    in features]), accumulated in fp32 and rounded once to ``out_dtype`` (bfloat16,
    float16 or float32).

    ``out`` may name a contiguous [M, N] tensor of dtype ``out_dtype`` to write into.
    K is at most 2^28.  Scale bytes that pad the last tile of a row have to be 0, as
    ``mxfp4_quantize`` and ``mxfp4_tile_scales`` write them.
    """
    if out is None:
        return _gemm(a, a_scales, b, b_scales, out_dtype)
    if out.dtype != out_dtype:
        raise ValueError(f"out must be {out_dtype}, got {out.dtype}")
    _gemm_out(out, a, a_scales, b, b_scales)
    return out


def mxfp4_tile_scales(scales: torch.Tensor) -> torch.Tensor:
    """Row-major scale bytes [rows, cols / 32] (uint8) -> the tiles that the operators
    take; what pads the last tiles is 0.  Plain torch, on any device."""
    if scales.dim() != 2 or scales.dtype != torch.uint8:
        raise ValueError("scales must be uint8 [rows, cols / 32]")
    rows, blocks = scales.shape
    tiles_m, tiles_k, _ = _tiles(rows, BLOCK * blocks)
    flat = scales.new_zeros((tiles_m * 128, tiles_k * 4))
    flat[:rows, :blocks] = scales
    # row = 32 * q + lane of its tile: byte lane * 16 + q * 4 + block
    tiled = flat.reshape(tiles_m, 4, 32, tiles_k, 4).permute(0, 3, 2, 1, 4)
    return tiled.reshape(tiles_m, tiles_k, 512).contiguous()


def mxfp4_untile_scales(tiles: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """The inverse of ``mxfp4_tile_scales``: scale bytes [rows, cols / 32] of a
    quantised [rows, cols] matrix."""
    if cols % BLOCK or tiles.dtype != torch.uint8 or tiles.shape != _tiles(rows, cols):
        raise ValueError(f"scales of a [{rows}, {cols}] matrix must be uint8 {_tiles(rows, cols)}, "
                         f"got {tiles.dtype} {tuple(tiles.shape)}")
    tiles_m, tiles_k, _ = tiles.shape
    flat = tiles.reshape(tiles_m, tiles_k, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return flat.reshape(tiles_m * 128, tiles_k * 4)[:rows, :cols // BLOCK].contiguous()
