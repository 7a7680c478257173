"""sandwich_rmsnorm on rows whose squares leave fp32's range: the largest and the
smallest numbers of bf16 and fp32, in every kernel behind the operator.

The formula is defined for them (rms(v) is of order 1 whatever the size of v), so
they are held to the same bounds as other rows: the scaling that brings the squares
back into range is by a power of two, which rounds nothing.  Inputs keep every value
that the formula forms away from fp32's subnormals, apart from squares.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import ops
from oracle.inputs import randn
from tests.conftest import to_device
from tests.test_sandwich_norm_cuda import check, make

pytestmark = pytest.mark.gpu

WIDE = ["float32", "bfloat16"]  # fp16's squares always fit fp32

# One shape for each way to hold a row: threads of a part of a warp (1 x 8 .. 16), of a
# warp, of several, of a whole block, a row on or off 16 bytes; the ring of one warp and
# of several per row, weights kept and read again, on and off 16 bytes; three passes.
SHAPES = [(5, 24), (5, 100), (3, 203), (9, 512), (4, 1001), (3, 2048), (2, 4099), (3, 8192),
          (2, 16384), (2, 32768), (700, 1024), (900, 1003), (300, 4096), (257, 8191), (64, 20480),
          (2, 40001), (2, 70000)]


def scaled(d, dtype, rows, **by):
    """Multiplies rows of x and residual, and whole weights, and rounds to dtype."""
    out = {}
    for k, v in d.items():
        f = np.float64(by.get(k, 1.0))
        w = v.astype(np.float64)
        if v.ndim == 2 and len(rows) < len(v):
            w[rows] *= f
        else:
            w *= f
        out[k] = ops.round_to(w.astype(np.float32), dtype)
        assert np.isfinite(out[k]).all()
    return out


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_large_x(shape, dtype):
    """|x| about 2^98 and 2^122: its squares are infinities, the branch is of order 1."""
    for e in (98, 122):
        d = make(shape, dtype, (shape[1],), seed=shape[1])
        check(scaled(d, dtype, range(shape[0]), x=2.0 ** e), dtype, alpha=0.75)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_large_h(shape, dtype):
    """The residual's squares, and so h's, are infinities; those of x as well or not."""
    for x in (1.0, 2.0 ** 100):
        d = make(shape, dtype, seed=shape[1])
        check(scaled(d, dtype, range(shape[0]), residual=2.0 ** 118, x=x), dtype)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_small_rows_without_eps(shape, dtype):
    """eps = 0: squares of x below fp32's smallest number, then those of h too (both
    parts of h brought down, the branch by its weight)."""
    d = make(shape, dtype, seed=shape[1])
    every = range(shape[0])
    check(scaled(d, dtype, every, x=2.0 ** -90), dtype, eps=0.0)
    check(scaled(d, dtype, every, residual=2.0 ** -80, post=2.0 ** -80), dtype, eps=0.0)
    check(scaled(d, dtype, every, x=2.0 ** -100, residual=2.0 ** -80, post=2.0 ** -80), dtype,
          eps=0.0)


@pytest.mark.parametrize("eps", [1e-30, 1e-36])
def test_small_eps_counts(eps):
    """Rows whose mean square is about eps, both far below the normal range of squares."""
    for shape in ((3, 203), (2, 4099), (700, 1024), (2, 70000)):
        d = make(shape, "float32", seed=3)
        check(scaled(d, "float32", range(shape[0]), x=float(np.sqrt(eps)),
                     residual=float(np.sqrt(eps)), post=float(np.sqrt(eps))), "float32", eps=eps)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("shape", [(37, 24), (37, 100), (37, 203), (37, 512), (37, 1001), (9, 4099),
                                   (700, 1024), (900, 1003), (300, 4096), (3, 70000)], ids=str)
def test_other_rows_keep_their_values(shape, dtype):
    """Rows out of range among others that share their warps, blocks and rings."""
    import torch

    rows = list(range(0, shape[0], 5))
    d = make(shape, dtype, (shape[1],), seed=1)
    want = check(d, dtype)
    got = check(scaled(d, dtype, rows, x=2.0 ** 110, residual=2.0 ** 90), dtype)
    keep = [r for r in range(shape[0]) if r % 5]
    for g, w in zip(got, want):
        assert torch.equal(g[keep], w[keep])


def test_zero_rows_without_eps_are_nan_and_alone():
    """0 / 0: NaN in a row of zeros with eps = 0, as the formula has it, in h only from x."""
    import torch

    import aot_kernel

    for shape in ((6, 24), (6, 512), (700, 1024), (3, 70000)):
        x, r = randn(shape, 1, "float32"), randn(shape, 2, "float32")
        x[2] = 0
        w = torch.ones(shape[1], device="cuda")
        out, h = aot_kernel.sandwich_rmsnorm(to_device(x, "float32"), to_device(r, "float32"), w, w, 0.0)
        for t in (out, h):
            assert torch.isnan(t[2]).all() and torch.isfinite(t[:2]).all() and torch.isfinite(t[3:]).all()


@pytest.mark.parametrize("shape", [(4, 512), (900, 1003), (2, 70000)], ids=str)
def test_infinities_among_large_values(shape):
    """One infinity in a row of large numbers: NaN there, and the rest of the branch 0."""
    import torch

    import aot_kernel

    x = randn(shape, 1, "float32") * np.float32(2.0 ** 100)
    r = randn(shape, 2, "float32")
    x[1, 7] = np.inf
    w = torch.ones(shape[1], device="cuda")
    out, h = aot_kernel.sandwich_rmsnorm(to_device(x, "float32"), to_device(r, "float32"), w, w)
    got = h[1].cpu().numpy()
    assert np.isnan(got[7]) and np.array_equal(np.delete(got, 7), np.delete(r[1], 7))
    assert torch.isnan(out[1]).all()
    assert torch.isfinite(h[0]).all() and torch.isfinite(out[0]).all()


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("cols", [24, 203, 1024, 1029, 40001])
@pytest.mark.parametrize("gate", ["row", "group", "full"])
def test_gates(gate, cols, dtype):
    B, S = (7, 150) if cols < 40000 else (2, 3)
    shape = {"row": (B, S, 1), "group": (B, 1, cols), "full": (B, S, cols)}[gate]
    d = make((B, S, cols), dtype, shape, seed=cols)
    d["x"] = ops.round_to(d["x"] * np.float32(2.0 ** 105), dtype)
    check(d, dtype, alpha=1.5)


@pytest.mark.parametrize("shape", [(40, 24), (40, 203), (40, 512), (40, 1001), (700, 1024), (900, 1003),
                                   (4, 70000)], ids=str)
def test_nan_rows_beside_rows_out_of_range(shape):
    """NaN stays in its row whatever its neighbours are; they are normalised as ever."""
    import torch

    import aot_kernel

    d = make(shape, "float32", seed=2)
    rows = list(range(1, shape[0], 3))
    d = scaled(d, "float32", rows, x=2.0 ** 110)
    bad = list(range(2, shape[0], 3))
    d["x"][bad, shape[1] // 2] = np.nan
    dev = {k: to_device(v, "float32") for k, v in d.items()}
    out, h = aot_kernel.sandwich_rmsnorm(dev["x"], dev["residual"], dev["post"], dev["pre"])
    assert torch.isnan(out[bad]).all() and torch.isnan(h[bad]).all()
    keep = [r for r in range(shape[0]) if r not in bad]
    good, h_good = check({k: v[keep] if v.ndim == 2 else v for k, v in d.items()}, "float32")
    # the rows that remain may be held by another kernel: sums in another order
    for a, b in ((out[keep], good), (h[keep], h_good)):
        assert (a - b).abs().max() <= 96 * 2.0 ** -23 * b.abs().max()


def test_two_graphs_of_rows_out_of_range():
    """Captured, and replayed at once on two streams with new inputs."""
    import torch

    import aot_kernel

    w = torch.ones(1003, device="cuda", dtype=torch.bfloat16)
    sets, graphs, got = [], [], []
    for e in (100, 60):
        x = to_device(ops.round_to(randn((900, 1003), e, "bfloat16") * np.float32(2.0 ** e), "bfloat16"),
                      "bfloat16")
        r = to_device(randn((900, 1003), e + 1, "bfloat16"), "bfloat16")
        sets.append((x, r))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(aot_kernel.sandwich_rmsnorm(x, r, w, w))
    for x, _ in sets:
        x.neg_()
        x[::7] *= 2.0 ** 20
    want = [aot_kernel.sandwich_rmsnorm(x, r, w, w) for x, r in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.isfinite(a[0]).all()
