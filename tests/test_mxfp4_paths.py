"""Every kernel behind mxfp4_gemm, at sizes that the rule in force sends to it.

CPU: the list below reaches each kernel, each width of the few-row kernel and each tile
width in one round and (where the rule ever has them) in several; so a later change of
the rule shows here what it left without a test.  GPU: the products of the list, exact in
all output types, on the kernel that the list names.
"""

from __future__ import annotations

import pytest

from aot_kernel import capi
from tests.test_mxfp4_cuda import check_exact

SMS = 148
TILES = {"pair_256": (2, 256), "pair_128": (2, 128), "one_128": (1, 128), "one_64": (1, 64)}

SHAPES = [
    # few rows, by the width that holds them: 16, 32, 64, 128
    (7, 3000, 2048, "split"), (16, 4096, 4096, "split"), (25, 5000, 1024, "split"),
    (32, 1001, 8192, "split"), (48, 4096, 4096, "split"), (40, 1001, 8192, "split"),
    (64, 512, 8192, "split"), (65, 2048, 8192, "split"), (100, 1024, 8192, "split"),
    (110, 4096, 14336, "split"), (128, 300, 16384, "split"), (90, 1001, 4096, "split"),
    (127, 1002, 8224, "split"),
    # tiles of one CTA
    (128, 6144, 512, "one_64"), (777, 1001, 1376, "one_64"), (200, 4094, 544, "one_64"),
    (128, 18944, 512, "one_128"), (300, 6000, 288, "one_128"), (640, 7360, 256, "one_128"),
    (64, 30001, 256, "one_128"), (300, 28480, 96, "one_128"),
    # pairs: one round, several, rows of C that start anywhere
    (300, 4096, 1024, "pair_128"), (2048, 1021, 288, "pair_128"), (1024, 4736, 512, "pair_128"),
    (1024, 4735, 256, "pair_128"), (1024, 4734, 256, "pair_128"), (2048, 4672, 320, "pair_128"),
    (2048, 2176, 544, "pair_256"), (2048, 4480, 256, "pair_256"), (1024, 4737, 256, "pair_256"),
    (1500, 12001, 96, "pair_256"),
]


def rounds(m, n, path):
    cg, bn = TILES[path]
    tiles = -(-m // (cg * 128)) * -(-n // bn)
    return -(-tiles // (SMS // cg))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rule_sends_each_size_to_its_kernel(shape):
    assert capi.mxfp4_gemm_path(*shape[:3], SMS) == shape[3]


def test_list_reaches_every_kernel():
    widths = {next(w for w in (16, 32, 64, 128) if m <= w) for m, _, _, p in SHAPES if p == "split"}
    assert widths == {16, 32, 64, 128}
    seen = {(p, min(rounds(m, n, p), 2)) for m, n, _, p in SHAPES if p != "split"}
    # 64-column tiles never take a second round: 128-column ones then need one
    assert seen == {("one_64", 1), ("one_128", 1), ("one_128", 2), ("pair_128", 1), ("pair_128", 2),
                    ("pair_256", 1), ("pair_256", 2)}
    for m in range(1, 2049, 37):
        for n in range(1, 40000, 611):
            if capi.mxfp4_gemm_path(m, n, 256, SMS) == "one_64":
                assert rounds(m, n, "one_64") == 1


def test_path_refusals():
    for bad in ((0, 8, 32, SMS), (8, 0, 32, SMS), (8, 8, 0, SMS), (8, 8, 32, 1), (-1, 8, 32, SMS)):
        with pytest.raises(capi.AotkError) as e:
            capi.mxfp4_gemm_path(*bad)
        assert e.value.status == capi.ERR_INVALID_ARGUMENT
    for bad in ((8, 8, 40, SMS), (8, 1 << 31, 32, SMS), (8, 8, (1 << 28) + 32, SMS)):
        with pytest.raises(capi.AotkError) as e:
            capi.mxfp4_gemm_path(*bad)
        assert e.value.status == capi.ERR_UNSUPPORTED


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product_on_each_kernel(shape, dtype):
    import torch

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != SMS or capi.mxfp4_gemm_path(*shape[:3], sms) == shape[3]
    check_exact(*shape[:3], dtype, seed=31)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[3] == "split" and s[0] > 32], ids=str)
def test_few_row_products_at_once_and_captured(shape):
    """The widths whose sums are received over the ring: many in flight on two streams,
    and a graph of them, against one alone."""
    import torch

    import aot_kernel
    from oracle.inputs import randn
    from tests.conftest import to_device

    M, N, K, _ = shape
    a = aot_kernel.mxfp4_quantize(to_device(randn((M, K), 1), "bfloat16"))
    b = aot_kernel.mxfp4_quantize(to_device(randn((N, K), 2), "bfloat16"))
    want = aot_kernel.mxfp4_gemm(*a, *b)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(aot_kernel.mxfp4_gemm(*a, *b))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [aot_kernel.mxfp4_gemm(*a, *b) for _ in range(4)]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got + kept)
    assert capi.watchdog_status() == 0
