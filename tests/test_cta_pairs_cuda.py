"""CTA-pair products back to back: the next launch's CTAs take over an SM as soon as one
of a pair leaves it, so nothing may be on its way to a CTA that has left.

Chains of the pair kernels (4-bit and 16-bit; one round of tiles and several, one and two
accumulators, rows on and off 16 bytes), with few-row products of other barrier layouts in
between, against each product alone.
"""

from __future__ import annotations

import pytest

from oracle.inputs import randn
from tests.conftest import to_device

pytestmark = pytest.mark.gpu


def products():
    import aot_kernel

    def mx(m, n, k, seed):
        a = aot_kernel.mxfp4_quantize(to_device(randn((m, k), seed), "bfloat16"))
        b = aot_kernel.mxfp4_quantize(to_device(randn((n, k), seed + 1), "bfloat16"))
        return lambda: aot_kernel.mxfp4_gemm(*a, *b)

    def wide(m, n, k, seed):
        a, b = to_device(randn((m, k), seed), "bfloat16"), to_device(randn((k, n), seed + 1), "bfloat16")
        return lambda: aot_kernel.gemm(a, b)

    return [mx(512, 4096, 256, 1), mx(8, 2048, 512, 3), mx(1024, 4736, 256, 5), mx(2048, 5000, 288, 7),
            mx(1024, 4737, 96, 9), wide(2048, 4096, 4096, 11), mx(100, 640, 256, 13),
            wide(4096, 6144, 4096, 15), mx(2304, 6144, 64, 17)]


def test_chains_of_pair_products():
    import torch

    from aot_kernel import capi

    steps = products()
    want = []
    for f in steps:
        want.append(f())
        torch.cuda.synchronize()
    for _ in range(20):
        got = [f() for f in steps + steps[::-1]]
        for g, w in zip(got, want + want[::-1]):
            assert torch.equal(g, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [f() for f in steps * 3]
    for _ in range(10):
        graph.replay()
        for i, g in enumerate(got):
            assert torch.equal(g, want[i % len(want)])
    assert capi.watchdog_status() == 0
