"""The 4-bit operators without a GPU: the oracle against the format's definition,
the scale layout, and what the wrappers and the C ABI refuse."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import aot_kernel
from aot_kernel import capi
from oracle import ops


def test_oracle_rounds_to_the_nearest_element():
    """Every element, every midpoint (to the even code) and both sides of it."""
    x = np.zeros((1, 32), np.float32)
    want = np.zeros(32, np.uint8)
    x[0, 31], want[31] = 6.0, 7  # fixes the scale at 2^0
    for i in range(7):
        mid = np.float32((ops.E2M1[i] + ops.E2M1[i + 1]) / 2)
        x[0, 4 * i:4 * i + 4] = (ops.E2M1[i], np.nextafter(mid, np.float32(0)), mid,
                                 np.nextafter(mid, np.float32(9)))
        want[4 * i:4 * i + 4] = (i, i, i + i % 2, i + 1)
    x[0, 28:31], want[28:31] = (-0.0, -5.0, 7.5), (8, 14, 7)
    code, scale = ops.mxfp4_quantize(x)
    assert scale.tolist() == [[127]] and code[0].tolist() == want.tolist()


def test_oracle_scales():
    x = np.zeros((1, 32 * 7), np.float32)
    for j, v in enumerate((0.0, 4.0, 7.99, 8.0, np.float32(2.0) ** -149, 3e38, np.nan)):
        x[0, 32 * j + 5] = v
    _, scale = ops.mxfp4_quantize(x)
    assert scale[0].tolist() == [0, 127, 127, 128, 0, 252, 255]


@pytest.mark.parametrize("rows,blocks", [(1, 1), (127, 3), (128, 4), (130, 5), (257, 9)])
def test_scale_tiles(rows, blocks):
    s = np.random.default_rng(rows).integers(0, 256, (rows, blocks), dtype=np.uint8)
    tiles = aot_kernel.mxfp4_tile_scales(torch.from_numpy(s))
    assert np.array_equal(tiles.numpy(), ops.mxfp4_tile(s))
    back = aot_kernel.mxfp4_untile_scales(tiles, rows, 32 * blocks)
    assert np.array_equal(back.numpy(), s)


def test_scale_tile_refusals():
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_tile_scales(torch.zeros(4, 4))
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_tile_scales(torch.zeros(4, dtype=torch.uint8))
    tiles = torch.zeros(1, 1, 512, dtype=torch.uint8)
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_untile_scales(tiles, 129, 32)
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_untile_scales(tiles, 4, 40)
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_untile_scales(tiles.float(), 4, 32)


def test_wrappers_refuse_cpu_tensors():
    u8 = dict(dtype=torch.uint8)
    codes, scales = torch.zeros(4, 16, **u8), torch.zeros(1, 1, 512, **u8)
    with pytest.raises(RuntimeError):
        aot_kernel.mxfp4_quantize(torch.zeros(4, 32))
    with pytest.raises(RuntimeError):
        aot_kernel.mxfp4_dequantize(codes, scales)
    with pytest.raises(RuntimeError):
        aot_kernel.mxfp4_gemm(codes, scales, codes, scales)
    w = torch.ones(8)
    with pytest.raises(ValueError):
        aot_kernel.sandwich_rmsnorm(torch.zeros(2, 8), torch.zeros(2, 8), w, w)


BF16, F32, I8 = capi.BFLOAT16, capi.FLOAT32, capi.INT8


@pytest.mark.parametrize("call,status", [
    (lambda: capi.mxfp4_quantize(16, 16, 16, 32, -1, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_quantize(16, 16, 16, 40, 4, 40, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_quantize(16, 16, 16, 32, 4, 32, I8), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_quantize(16, 16, None, 32, 4, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_quantize(16, 16, 16, 31, 4, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_quantize(24, 16, 16, 32, 4, 32, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_quantize(16, 16, 16, 32, 1 << 31, 32, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_dequantize(16, 16, None, 4, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_dequantize(16, 16, 16, 4, 33, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_dequantize(16, 16, 16, 4, 32, 9), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_gemm(16, 16, 16, 16, 16, 4, -4, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_gemm(16, 16, 16, 16, 16, 4, 4, 48, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_gemm(16, 16, 16, 16, 16, 4, 4, 32, I8), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_gemm(16, 16, 16, None, 16, 4, 4, 32, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_gemm(None, 16, 16, 16, 16, 4, 4, 0, BF16), capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.mxfp4_gemm(16, 16, 16, 24, 16, 4, 4, 32, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.mxfp4_gemm(16, 16, 16, 16, 16, 1 << 31, 4, 32, BF16), capi.ERR_UNSUPPORTED),
    (lambda: capi.sandwich_rmsnorm(16, 16, 16, 16, 16, 16, None, 0, 0, 1.0, -1, 8, 1e-6, BF16),
     capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.sandwich_rmsnorm(16, 16, 16, 16, None, 16, None, 0, 0, 1.0, 2, 8, 1e-6, BF16),
     capi.ERR_INVALID_ARGUMENT),
    (lambda: capi.sandwich_rmsnorm(16, 16, 16, 16, 16, 16, 16, 3, 8, 1.0, 4, 8, 1e-6, BF16),
     capi.ERR_INVALID_ARGUMENT),  # three gate rows for four rows
    (lambda: capi.sandwich_rmsnorm(16, 16, 16, 16, 16, 16, 16, 1, 4, 1.0, 4, 8, 1e-6, BF16),
     capi.ERR_INVALID_ARGUMENT),  # gate columns neither 1 nor 8
    (lambda: capi.sandwich_rmsnorm(16, 16, 16, 16, 16, 16, None, 0, 0, 1.0, 2, 8, 1e-6, I8),
     capi.ERR_UNSUPPORTED),
])
def test_c_abi_refusals(call, status):
    with pytest.raises(capi.AotkError) as exc:
        call()
    assert exc.value.status == status


def test_empty_problems_are_no_ops():
    capi.mxfp4_quantize(0, 0, 0, 0, 0, 64, BF16)
    capi.mxfp4_quantize(0, 0, 0, 0, 5, 0, F32)
    capi.mxfp4_dequantize(0, 0, 0, 0, 64, BF16)
    capi.mxfp4_gemm(0, 0, 0, 0, 0, 0, 8, 64, BF16)
    capi.mxfp4_gemm(0, 0, 0, 0, 0, 8, 0, 64, BF16)
    capi.sandwich_rmsnorm(0, 0, 0, 0, 0, 0, None, 0, 0, 1.0, 0, 64, 1e-6, BF16)


@pytest.mark.parametrize("K", [(1 << 28) + 32, 1 << 30, (1 << 31) - 256])
def test_product_refuses_sums_longer_than_its_waits(K):
    """Refused before any device is asked: a kernel's bounded waits would give up."""
    with pytest.raises(capi.AotkError) as e:
        capi.mxfp4_gemm(16, 16, 16, 16, 16, 4, 4, K, BF16)
    assert e.value.status == capi.ERR_UNSUPPORTED and "2^28" in str(e.value)
