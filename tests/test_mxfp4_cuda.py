"""Microscaled 4-bit quantisation and product on a B200 against the 64-bit oracle.

* Codes and scale bytes are determined, so they are compared byte for byte, and
  values read back are exact before their one rounding to the output type.
* The product of exact-sum inputs (elements are multiples of 1/2 and the scales
  lie within a few powers of two, so every partial sum is a multiple of the
  product of the two smallest scales / 4 and fits 24 bits) is compared bit for
  bit after the one rounding.  Elsewhere each of the at most K additions may be
  off by one unit in the last place of a partial sum, which sum |a| |b| bounds:
  |err| <= K 2^-23 (|A| |B|^T) + half a step of the output type.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import ops
from oracle.inputs import randn
from tests.conftest import to_device, torch_dtype

pytestmark = pytest.mark.gpu


def u8(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check_quantize(x, dtype, strided=0):
    """Compares mxfp4_quantize(x) with the oracle and returns (codes, scales)."""
    import aot_kernel

    rows, cols = x.shape
    if strided:
        wide = np.full((rows, cols + strided), np.nan, np.float32)
        wide[:, :cols] = x
        xd = to_device(wide, dtype)[:, :cols]
    else:
        xd = to_device(x, dtype)
    codes, scales = aot_kernel.mxfp4_quantize(xd)
    code, scale = ops.mxfp4_quantize(x)
    assert np.array_equal(codes.cpu().numpy(), ops.mxfp4_pack(code))
    assert np.array_equal(scales.cpu().numpy(), ops.mxfp4_tile(scale))
    return codes, scales


def check_dequantize(codes, scales, code, scale, dtype):
    import torch

    import aot_kernel

    got = aot_kernel.mxfp4_dequantize(codes, scales, torch_dtype(dtype))
    want = torch.from_numpy(ops.mxfp4_values(code, scale)).float().to(torch_dtype(dtype))
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=1.0), torch.nan_to_num(want, nan=1.0))


SHAPES = [(1, 32), (1, 4096), (3, 96), (127, 128), (128, 160), (130, 1056), (257, 4064), (33, 14336)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_quantize_and_read_back(shape, dtype):
    x = randn(shape, sum(shape), dtype, std=3.0)
    codes, scales = check_quantize(x, dtype)
    check_dequantize(codes, scales, *ops.mxfp4_quantize(x), dtype)


@pytest.mark.parametrize("extra", [1, 8, 96, 1024])
def test_quantize_strided_rows(extra, dtype):
    """Rows of a wider tensor; 1 and 8 leave rows that are not 16-byte aligned
    (fp16 / bf16 with 1, fp32 with 1)."""
    check_quantize(randn((70, 288), extra, dtype), dtype, strided=extra)


def test_quantize_unaligned_base(dtype):
    import torch

    import aot_kernel

    x = randn((5 * 64 + 1,), 3, dtype)
    xd = to_device(x, dtype)[1:].reshape(5, 64)  # contiguous, base off by one element
    codes, scales = aot_kernel.mxfp4_quantize(xd)
    code, scale = ops.mxfp4_quantize(x[1:].reshape(5, 64))
    assert np.array_equal(codes.cpu().numpy(), ops.mxfp4_pack(code))
    assert np.array_equal(scales.cpu().numpy(), ops.mxfp4_tile(scale))
    assert codes.dtype == torch.uint8


def test_quantize_midpoints_and_extremes(dtype):
    """Ties, values next to them, saturation, zeros of both signs, the type's
    largest and smallest numbers, infinities and NaN."""
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}[dtype]
    top = {"float32": 3.4e38, "float16": 65504.0, "bfloat16": 3.38e38}[dtype]
    rows = []
    for e in (0, 3, -9):
        r = np.zeros(32, np.float32)
        r[:7] = (ops.E2M1[:-1] + ops.E2M1[1:]) / 2
        r[7:15] = ops.E2M1
        r[15:22] = -r[:7]
        r[22:24] = (7.5, -7.75)
        rows.append(r * np.float32(2.0) ** e)
    for fill in (0.0, -0.0, tiny, -tiny, top, -top, np.inf, -np.inf, np.nan):
        r = np.zeros(32, np.float32)
        r[::3] = 1.0 if not np.isfinite(fill) or abs(fill) > 1 else 0.0
        r[13] = fill
        rows.append(r)
    x = ops.round_to(np.concatenate([np.stack(rows)] * 2, 1), dtype)
    codes, scales = check_quantize(x, dtype)
    check_dequantize(codes, scales, *ops.mxfp4_quantize(x), dtype)


def test_dequantize_every_code_and_scale(dtype):
    scale = np.arange(256, dtype=np.uint8).reshape(256, 1)
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    check_dequantize(u8(ops.mxfp4_pack(code)), u8(ops.mxfp4_tile(scale)), code, scale, dtype)


def test_quantize_empty():
    import torch

    import aot_kernel

    codes, scales = aot_kernel.mxfp4_quantize(torch.empty(0, 64, device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 1, 512)
    assert aot_kernel.mxfp4_dequantize(codes, scales).shape == (0, 64)
    codes, scales = aot_kernel.mxfp4_quantize(torch.empty(3, 0, device="cuda"))
    assert codes.shape == (3, 0) and scales.shape == (1, 0, 512)


# ---- product -------------------------------------------------------------------


def held(rows, cols, seed, spread):
    """Random codes and scale bytes within `spread` powers of two around 1."""
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    scale = (127 + rng.integers(-spread, spread + 1, (rows, cols // 32))).astype(np.uint8)
    return code, scale


def product(a, b, out_dtype, out=None):
    import aot_kernel

    return aot_kernel.mxfp4_gemm(u8(ops.mxfp4_pack(a[0])), u8(ops.mxfp4_tile(a[1])),
                                 u8(ops.mxfp4_pack(b[0])), u8(ops.mxfp4_tile(b[1])),
                                 torch_dtype(out_dtype), out=out)


def check_exact(M, N, K, out_dtype, seed=0, spread=1):
    import torch

    a, b = held(M, K, seed + M, spread), held(N, K, seed + N + 1, spread)
    av, bv = ops.mxfp4_values(*a), ops.mxfp4_values(*b)
    step = 2.0 ** (-2 * spread - 2)
    assert np.max(np.abs(av) @ np.abs(bv).T) < step * 2 ** 24  # every partial sum is exact
    want = torch.from_numpy(av @ bv.T).float().to(torch_dtype(out_dtype))
    got = product(a, b, out_dtype).cpu()
    assert got.shape == (M, N) and torch.equal(got, want)


GEMM_SHAPES = [
    (1, 1, 32), (1, 128, 4096), (2, 7, 64), (5, 1001, 96), (16, 256, 1376), (17, 130, 4096),
    (31, 384, 14336), (32, 512, 160), (48, 4096, 1024), (64, 640, 512), (65, 129, 288),
    (128, 1024, 2048), (129, 256, 256), (130, 100, 1056), (256, 512, 1024), (257, 257, 544),
    (384, 1280, 768), (777, 1001, 1376), (1024, 2048, 512),
    # more strips of 128 columns than clusters: several strips per cluster (M <= 32), one
    # CTA per strip, more strips than fit at once
    (3, 20001, 1056), (1, 24576, 2048), (20, 28700, 512), (70, 20000, 512), (2, 38001, 256),
    # several rounds of every tile width
    (1300, 5121, 320), (2100, 4352, 256), (700, 3584, 288), (192, 30000, 96),
]


@pytest.mark.parametrize("shape", GEMM_SHAPES, ids=str)
def test_gemm_exact(shape, dtype):
    check_exact(*shape, dtype)


@pytest.mark.parametrize("M", list(range(1, 20)) + [33, 47, 63, 95, 96, 97, 127, 160, 192, 255])
def test_gemm_every_small_m(M):
    check_exact(M, 264, 992, "bfloat16", seed=7)


@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 192, 224, 256, 288, 480, 512, 544, 1024, 2016])
@pytest.mark.parametrize("M", [3, 200])
def test_gemm_every_k_tail(M, K):
    check_exact(M, 320, K, "float32", seed=9)


@pytest.mark.parametrize("shape", [(4, 512, 4096), (200, 640, 4096)], ids=str)
def test_gemm_of_quantized_values(shape, dtype):
    """quantise -> product, scales as real data has them."""
    import torch

    import aot_kernel

    M, N, K = shape
    x = randn((M, K), 1, "bfloat16") * np.exp(randn((M, 1), 2, "float32"))
    x = ops.round_to(x * np.where(randn((1, K), 3, "float32") > 2.5, 20.0, 1.0), "bfloat16")
    w = randn((N, K), 4, "bfloat16", std=K ** -0.5)
    a = aot_kernel.mxfp4_quantize(to_device(x, "bfloat16"))
    b = aot_kernel.mxfp4_quantize(to_device(w, "bfloat16"))
    got = aot_kernel.mxfp4_gemm(*a, *b, torch_dtype(dtype)).double().cpu().numpy()
    av, bv = ops.mxfp4_values(*ops.mxfp4_quantize(x)), ops.mxfp4_values(*ops.mxfp4_quantize(w))
    want = av @ bv.T
    half = torch.finfo(torch_dtype(dtype)).eps / 2
    bound = K * 2.0 ** -23 * (np.abs(av) @ np.abs(bv).T) * (1 + half) + half * np.abs(want)
    if dtype == "float16":
        bound = bound + 2.0 ** -25  # half the smallest subnormal
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("M", [3, 150])
def test_gemm_extreme_scales(M):
    """Scale bytes from both ends whose products lie in fp32's range."""
    rng = np.random.default_rng(5)
    K, N = 256, 192
    code_a, code_b = held(M, K, 1, 0)[0], held(N, K, 2, 0)[0]
    sa = np.where(rng.random((M, K // 32)) < 0.5, 0, 1).astype(np.uint8)        # 2^-127, 2^-126
    sb = np.where(rng.random((N, K // 32)) < 0.5, 253, 254).astype(np.uint8)    # 2^126, 2^127
    av, bv = ops.mxfp4_values(code_a, sa), ops.mxfp4_values(code_b, sb)
    got = product((code_a, sa), (code_b, sb), "float32").double().cpu().numpy()
    assert np.array_equal(got, av @ bv.T)


@pytest.mark.parametrize("M", [5, 140])
def test_gemm_nan_scale_stays_in_its_row(M):
    K, N = 512, 200
    a, b = held(M, K, 3, 1), held(N, K, 4, 1)
    a[1][2, 9] = 255
    b[1][131, 4] = 255
    want = ops.mxfp4_values(*a) @ ops.mxfp4_values(*b).T
    got = product(a, b, "float32").double().cpu().numpy()
    assert np.isnan(got[2]).all() and np.isnan(got[:, 131]).all()
    ok = ~np.isnan(want)
    assert np.array_equal(np.isnan(got), ~ok) and np.array_equal(got[ok], want[ok])


@pytest.mark.parametrize("M", [4, 136])
def test_gemm_overflow_and_saturation(M):
    """Sums above fp16's range become infinities of the right sign."""
    K, N = 4096, 136
    code = np.full((M, K), 7, np.uint8)
    code[1] = 15
    scale = np.full((M, K // 32), 127, np.uint8)
    cb, sb = np.full((N, K), 7, np.uint8), np.full((N, K // 32), 127, np.uint8)
    got = product((code, scale), (cb, sb), "float16").cpu()
    want = np.full((M, N), np.inf)
    want[1] = -np.inf
    assert np.array_equal(got.double().numpy(), want)


@pytest.mark.parametrize("shape", [(6, 136, 512), (150, 136, 512), (6, 131, 512), (150, 131, 512)],
                         ids=str)
def test_gemm_out_rows_and_neighbours(shape, dtype):
    """`out` as a row slice of a larger buffer: the rows around it stay as they were."""
    import torch

    M, N, K = shape
    a, b = held(M, K, 11, 1), held(N, K, 12, 1)
    for before in (1, 8):
        buf = torch.full((M + before + 9, N), 7.0, dtype=torch_dtype(dtype), device="cuda")
        out = buf[before:before + M]
        assert product(a, b, dtype, out=out).data_ptr() == out.data_ptr()
        want = torch.from_numpy(ops.mxfp4_values(*a) @ ops.mxfp4_values(*b).T).float()
        assert torch.equal(out.cpu(), want.to(torch_dtype(dtype)))
        assert (buf[:before] == 7).all() and (buf[before + M:] == 7).all()


def test_gemm_empty():
    import torch

    import aot_kernel

    def pair(rows, cols):
        return (torch.zeros(rows, cols // 2, dtype=torch.uint8, device="cuda"),
                torch.zeros((rows + 127) // 128, (cols + 127) // 128, 512, dtype=torch.uint8,
                            device="cuda"))

    assert aot_kernel.mxfp4_gemm(*pair(0, 64), *pair(8, 64)).shape == (0, 8)
    assert aot_kernel.mxfp4_gemm(*pair(8, 64), *pair(0, 64)).shape == (8, 0)
    out = torch.full((3, 5), 9.0, dtype=torch.bfloat16, device="cuda")
    aot_kernel.mxfp4_gemm(*pair(3, 0), *pair(5, 0), out=out)
    assert (out == 0).all()  # an empty sum


def test_refusals():
    import torch

    import aot_kernel

    x = torch.zeros(4, 64, device="cuda")
    c, s = aot_kernel.mxfp4_quantize(x)
    for bad in (x.int(), x[:, :40], x[0], x.t(), torch.zeros(4, 128, device="cuda")[:, ::2],
                x[:1].expand(4, 64)):
        with pytest.raises(ValueError):
            aot_kernel.mxfp4_quantize(bad)
    for codes, scales in ((c.int(), s), (c, s.float()), (c[:, :8], s), (c, s[0]), (c[0], s),
                          (c, s.expand(2, 1, 512)), (c.t(), s), (c[:, ::2], s)):
        with pytest.raises(ValueError):
            aot_kernel.mxfp4_dequantize(codes, scales)
        with pytest.raises(ValueError):
            aot_kernel.mxfp4_gemm(codes, scales, c, s)
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_dequantize(c, s, torch.int32)
    c2, s2 = aot_kernel.mxfp4_quantize(torch.zeros(4, 96, device="cuda"))
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_gemm(c, s, c2, s2)
    with pytest.raises(ValueError):
        aot_kernel.mxfp4_gemm(c, s, c, s, torch.float64)
    for out in (torch.empty(4, 5, device="cuda", dtype=torch.bfloat16),
                torch.empty(4, 4, device="cuda"), torch.empty(4, 4, dtype=torch.bfloat16),
                torch.empty(4, 8, device="cuda", dtype=torch.bfloat16)[:, ::2]):
        with pytest.raises(ValueError):
            aot_kernel.mxfp4_gemm(c, s, c, s, out=out)
    with pytest.raises(RuntimeError):
        aot_kernel.mxfp4_gemm(c, s, c.cpu(), s)


# ---- streams, graphs, a run of the operators together -----------------------------


@pytest.mark.parametrize("M", [7, 300])
def test_side_stream_and_graph(M):
    """On another stream, and captured once and replayed with new inputs."""
    import torch

    import aot_kernel

    K, N = 768, 520
    w = aot_kernel.mxfp4_quantize(to_device(randn((N, K), 2), "bfloat16"))
    xs = [to_device(randn((M, K), 20 + i), "bfloat16") for i in range(3)]

    def step(x):
        q = aot_kernel.mxfp4_quantize(x)
        return aot_kernel.mxfp4_gemm(*q, *w), aot_kernel.mxfp4_dequantize(*q)

    want = [step(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, want[0]))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want[i]))


def test_two_streams_at_once():
    """Products of every kernel on two streams, many in flight, against one alone."""
    import torch

    import aot_kernel

    K = 1024
    work = []
    for j, (M, N) in enumerate(((1, 2048), (40, 4096), (120, 640), (300, 2048), (1000, 1500))):
        a = aot_kernel.mxfp4_quantize(to_device(randn((M, K), j), "bfloat16"))
        b = aot_kernel.mxfp4_quantize(to_device(randn((N, K), 50 + j), "bfloat16"))
        work.append((a, b, aot_kernel.mxfp4_gemm(*a, *b)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for r in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                for a, b, want in work[:: 1 - 2 * k]:
                    got.append((aot_kernel.mxfp4_gemm(*a, *b), want))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in got)
    from aot_kernel import capi

    assert capi.watchdog_status() == 0


def test_offsets_beyond_32_bits():
    """More than 2^31 elements in x, in the values read back and in the product."""
    import torch

    import aot_kernel

    gen = torch.Generator(device="cuda").manual_seed(3)
    rows, cols = 65700, 32768
    x = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.bfloat16)
    codes, scales = aot_kernel.mxfp4_quantize(x)
    back = aot_kernel.mxfp4_dequantize(codes, scales)
    for r0 in (0, 65536 - 128, 65536 + 128 - 128):
        part = x[r0:r0 + 128].contiguous()
        c, s = aot_kernel.mxfp4_quantize(part)
        assert torch.equal(codes[r0:r0 + 128], c) and torch.equal(scales[r0 // 128], s[0])
        assert torch.equal(back[r0:r0 + 128], aot_kernel.mxfp4_dequantize(c, s))
    del x, back, codes, scales
    M, N, K = 65700, 32896, 64
    a = aot_kernel.mxfp4_quantize(torch.randn(M, K, generator=gen, device="cuda"))
    b = aot_kernel.mxfp4_quantize(torch.randn(N, K, generator=gen, device="cuda"))
    out = aot_kernel.mxfp4_gemm(*a, *b)
    av, bv = (aot_kernel.mxfp4_dequantize(*q, torch.float32) for q in (a, b))
    for r0 in (0, 65600):  # sums of 64 products of a few bits each: exact in fp32
        want = (av[r0:r0 + 64].double() @ bv.double().t()).float().to(torch.bfloat16)
        assert torch.equal(out[r0:r0 + 64], want)


@pytest.mark.parametrize("M", [1, 9, 260])
def test_block_in_four_bits(M):
    """One gated MLP block served in 4 bits between its norms: quantise, gate/up
    product, silu(gate) * up, quantise, down product, sandwich norm - each step
    against the oracle on the inputs that it was given."""
    import torch

    import aot_kernel

    H, I, eps = 512, 1376, 1e-6
    t = lambda shape, seed, std=1.0, mean=0.0: to_device(  # noqa: E731
        randn(shape, seed, "bfloat16", mean, std), "bfloat16")
    np64 = lambda v: v.detach().double().cpu().numpy()  # noqa: E731
    x, residual = t((M, H), 1), t((M, H), 2)
    w_gu, w_d = t((2 * I, H), 3, H ** -0.5), t((H, I), 4, I ** -0.5)
    post, pre, gate = t((H,), 5, 0.1, 1.0), t((H,), 6, 0.1, 1.0), t((H,), 7, 0.3)
    q_gu, q_d = aot_kernel.mxfp4_quantize(w_gu), aot_kernel.mxfp4_quantize(w_d)

    q_x = aot_kernel.mxfp4_quantize(x)
    gu = aot_kernel.mxfp4_gemm(*q_x, *q_gu)
    act = aot_kernel.silu_mul(gu[:, :I], gu[:, I:])
    q_a = aot_kernel.mxfp4_quantize(act)
    down = aot_kernel.mxfp4_gemm(*q_a, *q_d)
    out, h = aot_kernel.sandwich_rmsnorm(down, residual, post, pre, eps, gate=gate,
                                         residual_scale=0.5)

    def values(v):
        return ops.mxfp4_values(*ops.mxfp4_quantize(np64(v).astype(np.float32)))

    def close(got, a, b):
        want, bound = a @ b.T, 2.0 ** -23 * a.shape[1] * (np.abs(a) @ np.abs(b).T)
        assert np.all(np.abs(np64(got) - want) <= 1.01 * bound + 2.0 ** -8 * np.abs(want))

    close(gu, values(x), values(w_gu))
    close(down, values(act), values(w_d))
    o, hh, _ = ops.sandwich_rmsnorm(np64(down), np64(residual), np64(post), np64(pre), eps,
                                    np64(gate), 0.5)
    # fp32 work on values of order 1 and one rounding to bf16
    assert np.all(np.abs(np64(h) - hh) <= 2.0 ** -8 * np.abs(hh) + 1e-5)
    assert np.all(np.abs(np64(out) - o) <= 2.0 ** -8 * np.abs(o) + 1e-4)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("M,N,K", [(2, 40, 1 << 20), (130, 40, 1 << 20), (3, (1 << 20) + 5, 64),
                                   (130, (1 << 19) + 8, 64), ((1 << 20) + 3, 24, 96)], ids=str)
def test_gemm_long_sums_and_many_rows(M, N, K):
    """Elements 0, +-.5 and +-1 at scale 1: any partial sum is a multiple of 1/4 and at
    most K <= 2^20, so fp32 sums are exact in any order (22 bits)."""
    import torch

    import aot_kernel

    gen = torch.Generator(device="cuda").manual_seed(M)
    element = torch.tensor([0.0, 0.5, 1.0, -0.5, -1.0], device="cuda")
    code = torch.tensor([0, 1, 2, 9, 10], device="cuda", dtype=torch.uint8)

    def operand(rows):
        pick = torch.randint(0, 5, (rows, K), generator=gen, device="cuda")
        codes = code[pick[:, ::2]] | code[pick[:, 1::2]] << 4
        one = torch.full((rows, K // 32), 127, dtype=torch.uint8, device="cuda")
        return (codes, aot_kernel.mxfp4_tile_scales(one)), element[pick]

    a, av = operand(M)
    b, bv = operand(N)
    got = aot_kernel.mxfp4_gemm(*a, *b, torch.float32)
    for r in range(0, M, 1 << 17):  # bounds the 64-bit temporaries
        want = av[r:r + (1 << 17)].double() @ bv.double().t()
        assert torch.equal(got[r:r + (1 << 17)].double(), want)


@pytest.mark.parametrize("M", [5, 90, 300])
def test_gemm_of_a_matrix_with_itself(M):
    import torch

    import aot_kernel

    q, s = aot_kernel.mxfp4_quantize(to_device(randn((M, 320), M), "bfloat16"))
    got = aot_kernel.mxfp4_gemm(q, s, q, s, torch.float32)
    assert torch.equal(got, aot_kernel.mxfp4_gemm(q, s, q.clone(), s.clone(), torch.float32))
    v = aot_kernel.mxfp4_dequantize(q, s, torch.float32).double()
    # K = 320 additions, each off by at most one unit in the last place of sum |a| |b|
    assert ((got.double() - v @ v.t()).abs() <= 320 * 2.0 ** -23 * (v.abs() @ v.abs().t())).all()


def test_two_graphs_replayed_at_once():
    """The products keep no workspace that two graphs could share."""
    import torch

    import aot_kernel

    K, N = 2048, 1024
    w = aot_kernel.mxfp4_quantize(to_device(randn((N, K), 1), "bfloat16"))
    xs = [aot_kernel.mxfp4_quantize(to_device(randn((M, K), 2 + M), "bfloat16")) for M in (6, 6, 100, 200)]
    want = [aot_kernel.mxfp4_gemm(*x, *w) for x in xs]
    graphs, got = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append([aot_kernel.mxfp4_gemm(*x, *w) for _ in range(3)])
    streams = [torch.cuda.Stream() for _ in xs]
    for g in got:
        for t in g:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, v) for g, v in zip(got, want) for t in g)


FIRST_CALL = """
import torch, aot_kernel
gen = torch.Generator(device="cuda").manual_seed(1)
M, N, K = {M}, 264, 512
x = torch.randn(M, K, generator=gen, device="cuda", dtype=torch.bfloat16)
y = torch.randn(N, K, generator=gen, device="cuda", dtype=torch.bfloat16)
r = torch.randn(M, N, generator=gen, device="cuda", dtype=torch.bfloat16)
w = torch.ones(N, device="cuda", dtype=torch.bfloat16)
def step():
    a, b = aot_kernel.mxfp4_quantize(x), aot_kernel.mxfp4_quantize(y)
    c = aot_kernel.mxfp4_gemm(*a, *b)
    return c, aot_kernel.mxfp4_dequantize(*a), *aot_kernel.sandwich_rmsnorm(c, r, w, w)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
assert all(torch.equal(g, v) for g, v in zip(got, step()))
print("replayed")
"""


@pytest.mark.parametrize("M", [4, 70, 2500])
def test_first_call_may_be_captured(M):
    """No call is needed before a capture (in a process of its own: nothing is loaded)."""
    import os
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST_CALL.format(M=M)], capture_output=True,
                          text=True, timeout=300,
                          env=dict(os.environ, PYTHONPATH=os.pathsep.join(filter(None, sys.path))))
    assert done.returncode == 0 and "replayed" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("N", [1, 2, 3, 31, 66, 127, 130, 190, 1002, 1004])
@pytest.mark.parametrize("start", [0, 1, 2, 4, 8])
def test_gemm_rows_that_start_anywhere(N, start, dtype):
    """`out` from element `start` of a buffer on, rows of N elements, ragged last rows;
    what lies before and behind stays as it was."""
    import torch

    for M, K in ((139, 96), (300, 64), (9, 64)):
        a, b = held(M, K, 21, 1), held(N, K, 22, 1)
        buf = torch.full((start + M * N + 64,), 7.0, dtype=torch_dtype(dtype), device="cuda")
        product(a, b, dtype, out=buf[start:start + M * N].view(M, N))
        want = torch.from_numpy(ops.mxfp4_values(*a) @ ops.mxfp4_values(*b).T).float()
        got = buf.cpu()
        assert torch.equal(got[start:start + M * N].view(M, N), want.to(torch_dtype(dtype)))
        assert (got[:start] == 7).all() and (got[start + M * N:] == 7).all()


@pytest.mark.parametrize("M", [1, 30, 60, 128, 400])
def test_operands_written_by_the_kernel_before(M):
    """The weight is quantised by the launch right before the product that reads it."""
    import torch

    import aot_kernel

    K, N = 1024, 4096
    x = aot_kernel.mxfp4_quantize(to_device(randn((M, K), 1), "bfloat16"))
    ws = [to_device(randn((N, K), 2 + i), "bfloat16") for i in range(3)]
    want = []
    for w in ws:
        q = aot_kernel.mxfp4_quantize(w)
        torch.cuda.synchronize()
        want.append(aot_kernel.mxfp4_gemm(*x, *q))
        torch.cuda.synchronize()
    w = torch.empty_like(ws[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = aot_kernel.mxfp4_gemm(*x, *aot_kernel.mxfp4_quantize(w))
    for _ in range(10):
        for i, v in enumerate(ws):
            w.copy_(v)
            assert torch.equal(aot_kernel.mxfp4_gemm(*x, *aot_kernel.mxfp4_quantize(w)), want[i])
            graph.replay()
            assert torch.equal(got, want[i])
