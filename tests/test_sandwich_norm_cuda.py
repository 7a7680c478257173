"""The norms around a block (sandwich_rmsnorm) on a B200 against the 64-bit oracle.

Bounds, with u = 2^-24 and c steps of fp32 rounding behind a value (a thread's
share of a sum, the warp and block tree, the root, the products; a thread adds at
most max(64, cols / 256) squares):
  h:   |err| <= E_h = c u (|alpha residual| + |branch|), then half a step of h;
  out: the row's root mean square is off by at most c u plus rms(E_h) / rms(h)
       relative, so |err| <= |pre| / rms(h) (E_h + |h| (c u + rms(E_h) / rms(h))),
       then half a step of out.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import ops
from oracle.inputs import randn
from tests.conftest import to_device, torch_dtype

pytestmark = pytest.mark.gpu

EPS = 1e-6
SUBNORMAL = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}


def make(shape, dtype, gate_shape=None, seed=0):
    H = shape[-1]
    d = {
        "x": randn(shape, seed + 1, dtype, std=3.0),
        "residual": randn(shape, seed + 2, dtype),
        "post": randn((H,), seed + 3, dtype, mean=1.0, std=0.2),
        "pre": randn((H,), seed + 4, dtype, mean=1.0, std=0.2),
    }
    if gate_shape is not None:
        d["gate"] = randn(gate_shape, seed + 5, dtype, std=0.5)
    return d


def check(d, dtype, eps=EPS, alpha=1.0):
    import torch

    import aot_kernel

    dev = {k: to_device(v, dtype) for k, v in d.items()}
    out, h = aot_kernel.sandwich_rmsnorm(dev["x"], dev["residual"], dev["post"], dev["pre"], eps,
                                         gate=dev.get("gate"), residual_scale=alpha)
    assert out.shape == h.shape == d["x"].shape and out.dtype == h.dtype == torch_dtype(dtype)
    o, hh, branch = ops.sandwich_rmsnorm(d["x"], d["residual"], d["post"], d["pre"], eps,
                                         d.get("gate"), float(np.float32(alpha)))
    c = (max(64, d["x"].shape[-1] / 256) + 32) * 2.0 ** -24
    half, tiny = torch.finfo(torch_dtype(dtype)).eps / 2, SUBNORMAL[dtype] / 2
    e_h = c * (np.abs(alpha * d["residual"]) + np.abs(branch))
    rms = np.sqrt(np.mean(hh * hh, -1, keepdims=True) + eps)
    off = c + np.sqrt(np.mean(e_h * e_h, -1, keepdims=True)) / rms
    e_o = np.abs(d["pre"]) / rms * (e_h + np.abs(hh) * off)
    got_h, got_o = (v.double().cpu().numpy() for v in (h, out))
    assert np.all(np.abs(got_h - hh) <= (e_h + half * np.abs(hh)) * (1 + half) + tiny)
    assert np.all(np.abs(got_o - o) <= (e_o + half * np.abs(o)) * (1 + half) + tiny)
    return out, h


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 64, 255, 256, 1000, 1024, 2047, 2048, 4096, 4100,
                                  8192, 9001, 16384, 20000, 32768, 40001, 65536])
def test_row_lengths(cols, dtype):
    check(make((3, cols), dtype, (cols,), seed=cols), dtype)


@pytest.mark.parametrize("rows", [1, 2, 9, 149, 700])
def test_row_counts(rows, dtype):
    check(make((rows, 512), dtype, seed=rows), dtype, alpha=0.5)


@pytest.mark.parametrize("cols", [256, 511, 512, 777, 1000, 1160, 2047, 2049, 4096, 4099, 5120, 6001,
                                  8189, 8191, 8192, 9999, 12296, 16371, 16383, 16384])
def test_many_rows(cols, dtype):
    """Enough rows for every group of the streaming kernel to go round its ring, with
    a last row that ends inside a vector where the length is odd."""
    size = 4 if dtype == "float32" else 2
    rows = 2 * (3 << 20) // (cols * size) | 1
    d = make((rows, cols), dtype, (cols,), seed=cols)
    out, h = check(d, dtype, alpha=0.75)
    again, h2 = check({k: v[-5:] if v.ndim == 2 else v for k, v in d.items()}, dtype, alpha=0.75)
    for a, b in ((out[-5:], again), (h[-5:], h2)):  # two orders of the sums
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -6 * b.double().abs().max()


@pytest.mark.parametrize("cols", [1024, 1029])
@pytest.mark.parametrize("gate", ["none", "row", "group", "full"])
def test_many_rows_gates(gate, cols, dtype):
    B, S = 7, 300
    shape = {"none": None, "row": (B, S, 1), "group": (B, 1, cols), "full": (B, S, cols)}[gate]
    check(make((B, S, cols), dtype, shape, seed=cols), dtype, alpha=1.5)


GATES = [None, (48,), (1,), (1, 1, 48), (4, 1, 48), (4, 5, 1), (4, 1, 1), (4, 5, 48)]


@pytest.mark.parametrize("cols", [48, 35])
@pytest.mark.parametrize("gate", GATES, ids=str)
def test_gate_shapes(gate, cols, dtype):
    g = None if gate is None else gate[:-1] + (cols if gate[-1] == 48 else 1,)
    check(make((4, 5, cols), dtype, g), dtype, alpha=1.25)


@pytest.mark.parametrize("alpha", [0.0, 1.0, -2.5, 0.1])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-2])
def test_scales(alpha, eps):
    check(make((17, 640), "float32", (17, 1)), "float32", eps=eps, alpha=alpha)


def test_agrees_with_add_rmsnorm_of_the_normed_branch():
    """With no gate, h and out are those of rmsnorm then add_rmsnorm up to the
    roundings in between."""
    import torch

    import aot_kernel

    d = {k: to_device(v, "float32") for k, v in make((50, 1024), "float32").items()}
    out, h = aot_kernel.sandwich_rmsnorm(d["x"], d["residual"], d["post"], d["pre"], EPS)
    branch = aot_kernel.rmsnorm(d["x"], d["post"], EPS)
    out2, h2 = aot_kernel.add_rmsnorm(branch, d["residual"], d["pre"], EPS)
    # each side has at most 96 fp32 roundings behind a value of order 10
    assert torch.allclose(h, h2, rtol=0, atol=2 * 96 * 2.0 ** -24 * 16)
    assert torch.allclose(out, out2, rtol=0, atol=4 * 96 * 2.0 ** -24 * 16)


def test_zero_rows_and_nan_rows(dtype):
    """A row of zeros gives zeros, and a NaN or an infinity stays in its row."""
    import torch

    import aot_kernel

    d = make((6, 264), dtype, (264,))
    d["x"][1] = 0
    d["residual"][1] = 0
    d["x"][2, 5] = np.nan
    d["residual"][4, 7] = np.inf
    dev = {k: to_device(v, dtype) for k, v in d.items()}
    out, h = aot_kernel.sandwich_rmsnorm(dev["x"], dev["residual"], dev["post"], dev["pre"], EPS,
                                         gate=dev["gate"])
    assert (out[1] == 0).all() and (h[1] == 0).all()
    assert torch.isnan(out[2]).all() and torch.isnan(h[2]).all()
    assert torch.isinf(h[4, 7]) and torch.isfinite(h[4]).sum() == 263
    assert torch.isnan(out[4, 7]) and (out[4].nan_to_num(nan=0.0) == 0).all()
    keep = [0, 3, 5]
    alone, h_alone = check({k: (v[keep] if v.shape[:1] == (6,) else v) for k, v in d.items()}, dtype)
    assert torch.equal(out[keep], alone) and torch.equal(h[keep], h_alone)


def test_large_values():
    """Squares of fp16's and bf16's largest numbers stay within fp32."""
    d = make((2, 2048), "float16")
    d["x"][:] = np.where(d["x"] < 0, -65504.0, 65504.0)
    check(d, "float16")


def test_unaligned_base(dtype):
    import torch

    import aot_kernel

    d = {k: to_device(v, dtype) for k, v in make((5, 256), dtype).items()}
    want = aot_kernel.sandwich_rmsnorm(d["x"], d["residual"], d["post"], d["pre"], EPS)
    flat = torch.empty(5 * 256 + 1, dtype=d["x"].dtype, device="cuda")
    x = flat[1:].reshape(5, 256)
    x.copy_(d["x"])
    got = aot_kernel.sandwich_rmsnorm(x, d["residual"], d["post"], d["pre"], EPS)
    eps = torch.finfo(d["x"].dtype).eps  # sums in another order: one step of the type
    for g, w in zip(got, want):
        assert torch.allclose(g.double(), w.double(), rtol=2 * max(eps, 96 * 2.0 ** -24), atol=1e-6)


def test_empty():
    import torch

    import aot_kernel

    w = torch.ones(8, device="cuda")
    e = torch.empty(0, 8, device="cuda")
    out, h = aot_kernel.sandwich_rmsnorm(e, e, w, w)
    assert out.shape == h.shape == (0, 8)
    e = torch.empty(3, 0, device="cuda")
    out, h = aot_kernel.sandwich_rmsnorm(e, e, w[:0], w[:0], gate=w[:0])
    assert out.shape == (3, 0)


def test_refusals():
    import torch

    import aot_kernel

    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    f = aot_kernel.sandwich_rmsnorm
    for args, kw in (
        ((x, x[:2], w, w), {}), ((x, x.half(), w, w), {}), ((x, x, w.half(), w), {}),
        ((x.t(), x.t(), w, w), {}), ((x, x, w, w), {"gate": w[:4]}),
        ((x, x, w, w), {"gate": w.half()}), ((x, x, w, w), {"gate": torch.ones(2, 8, device="cuda")}),
        ((x, x, w, w), {"gate": torch.ones(8, 2, device="cuda").t()[:1]}),
        ((x, x, w, w.cpu()), {}),
    ):
        with pytest.raises(ValueError):
            f(*args, **kw)
    for weights in ((w[:4], w), (w, w[:4]), (x, w)):
        with pytest.raises(ValueError):
            f(x, x, *weights)
    with pytest.raises(ValueError):
        f(x.double(), x.double(), w.double(), w.double())


@pytest.mark.parametrize("shape", [(), (3, 8), (1, 3, 8), (2, 3, 4), (4,), (1, 2, 3, 8), (3, 1),
                                   (3, 1, 8)])
def test_gate_refusals(shape):
    import torch

    import aot_kernel

    x, w = torch.zeros(2, 3, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError):
        aot_kernel.sandwich_rmsnorm(x, x, w, w, gate=torch.ones(shape, device="cuda"))


def test_outputs_take_no_part_in_autograd():
    import torch

    import aot_kernel

    x = torch.randn(4, 64, device="cuda")
    w = torch.nn.Parameter(torch.ones(64, device="cuda"))
    out, h = aot_kernel.sandwich_rmsnorm(x, x, w, w, gate=w)
    assert not out.requires_grad and not h.requires_grad


def test_stream_and_graph():
    import torch

    import aot_kernel

    d = {k: to_device(v, "bfloat16") for k, v in make((33, 1024), "bfloat16", (33, 1)).items()}

    def step():
        return aot_kernel.sandwich_rmsnorm(d["x"], d["residual"], d["post"], d["pre"], EPS,
                                           gate=d["gate"], residual_scale=0.7)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    d["x"].neg_()
    graph.replay()
    new = step()
    assert all(torch.equal(a, b) for a, b in zip(got, new))
    assert not torch.equal(got[0], want[0])


@pytest.mark.parametrize("cols", [16384, 8191])
def test_offsets_beyond_32_bits(cols):
    import torch

    import aot_kernel

    rows = (1 << 31) // cols + 300
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.bfloat16)
    residual = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.bfloat16)
    post, pre = (torch.randn(cols, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    gate = torch.randn(rows, 1, generator=gen, device="cuda", dtype=torch.bfloat16)
    out, h = aot_kernel.sandwich_rmsnorm(x, residual, post, pre, EPS, gate=gate)
    for r0 in (0, rows - 9):
        part = [t[r0:r0 + 9].clone() for t in (x, residual, gate)]
        o, hh = aot_kernel.sandwich_rmsnorm(part[0], part[1], post, pre, EPS, gate=part[2])
        for g, w in ((out, o), (h, hh)):  # sums in another order: at most one step of bf16
            g = g[r0:r0 + 9].double()
            assert ((g - w.double()).abs() <= 2.0 ** -7 * w.double().abs() + 1e-3).all()


@pytest.mark.parametrize("shape", [(3, 100), (5, 512), (700, 1000), (700, 2048), (3, 40000)], ids=str)
def test_one_tensor_in_every_place(shape):
    """x is the residual and the gate too, and one weight serves both norms."""
    d = make(shape, "bfloat16")
    d["residual"] = d["gate"] = d["x"]
    d["pre"] = d["post"]
    import torch

    import aot_kernel

    x, w = to_device(d["x"], "bfloat16"), to_device(d["post"], "bfloat16")
    out, h = aot_kernel.sandwich_rmsnorm(x, x, w, w, EPS, gate=x)
    o2, h2 = check(d, "bfloat16")
    assert torch.equal(out, o2) and torch.equal(h, h2)


@pytest.mark.parametrize("cols", [1000, 1003])
def test_graph_of_many_rows(cols):
    """Captured and replayed with new inputs; two replays in flight on two streams."""
    import torch

    import aot_kernel

    sets = [{k: to_device(v, "bfloat16") for k, v in make((900, cols), "bfloat16", (900, 1), s).items()}
            for s in (10, 20)]

    def step(d):
        return aot_kernel.sandwich_rmsnorm(d["x"], d["residual"], d["post"], d["pre"], EPS,
                                           gate=d["gate"])

    graphs, got = [], []
    for d in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(step(d))
    for d in sets:
        d["x"].neg_()
    want = [step(d) for d in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("cols", [1, 2, 3, 5, 7, 9, 11, 13, 15, 17, 2045])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 7, 8, 33])
def test_tensor_ends_anywhere_in_a_vector(rows, cols, dtype):
    check(make((rows, cols), dtype, (1, cols), rows + cols), dtype)


@pytest.mark.parametrize("gate", ["none", "channel", "group"])
@pytest.mark.parametrize("cols", [9000, 10240, 16392, 20480, 24568, 24584])
def test_many_long_rows(cols, gate, dtype):
    shape = {"none": None, "channel": (1, cols), "group": (12, 1, cols)}[gate]
    check(make((12, 27, cols), dtype, shape, cols), dtype, alpha=0.7)


@pytest.mark.parametrize("cols", [4096, 1001, 20480, 640])
def test_residual_written_by_the_kernel_before(cols):
    """A chain of norms, each reading what the one before has just written (eagerly and
    captured, with nothing between the launches), against the same chain with waits."""
    import torch

    import aot_kernel

    d = {k: to_device(v, "bfloat16") for k, v in make((600, cols), "bfloat16").items()}

    def chain(wait):
        x, h, kept = d["x"], d["residual"], []
        for _ in range(6):
            x, h = aot_kernel.sandwich_rmsnorm(x, h, d["post"], d["pre"], EPS, residual_scale=0.9)
            kept += [x, h]
            if wait:
                torch.cuda.synchronize()
        return kept

    want = chain(True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(False)
    for _ in range(5):
        for t in got:
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
