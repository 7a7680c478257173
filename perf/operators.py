"""Workloads of the 4-bit linear path: microscaled quantisation, its product
and the two norms around a block, in plain torch and through the package.

Formulas (MX format: blocks of 32 along the row share a power-of-two scale,
elements are e2m1):

* quantise and read back: per block, S = 2^(floor(log2 max|x|) - 2), element
  q = x / S rounded to the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} (ties to the
  even code, larger magnitudes to 6), value q * S;
* product: C[m, n] = sum_k A[m, k] B[n, k] over the values that the codes and
  scales of both stand for, fp32 accumulation, one rounding;
* sandwich norm: h = alpha * residual + gate * (rms(x) * post_weight),
  y = rms(h) * pre_weight, with rms(v) = v / sqrt(mean(v^2) + eps).

`own` chooses between the plain form (False) and the package's operators.
"""

import functools
import os
import sys

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


@functools.lru_cache(maxsize=1)
def _api():
    path = os.path.join(os.getcwd(), "inference-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import aot_kernel

    return aot_kernel


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # One decoded token's activations before a 4-bit projection.
        {"name": "quant_token", "op": "quant", "rows": 1, "cols": 4096, "pad": 0, "dtype": "bf16"},
        # A prefill batch at the width of the tensor-parallel MLP block.
        {"name": "quant_prefill", "op": "quant", "rows": 4096, "cols": 8192, "pad": 0,
         "dtype": "bf16"},
        # The gate half of a fused gate/up output (strided rows), an odd number of
        # rows, a width that ends inside a 128-column scale tile, fp16.
        {"name": "quant_strided", "op": "quant", "rows": 1237, "cols": 11040, "pad": 11040,
         "dtype": "fp16"},
        # A weight matrix converted from fp32.
        {"name": "quant_weight", "op": "quant", "rows": 14336, "cols": 4096, "pad": 0,
         "dtype": "fp32"},
        # One token through the fused gate/up projection: the weight stream.
        {"name": "gemm_token", "op": "gemm", "m": 1, "n": 28672, "k": 4096, "dtype": "bf16"},
        # A decode batch through the down projection: few output columns, long K.
        {"name": "gemm_decode", "op": "gemm", "m": 48, "n": 4096, "k": 14336, "dtype": "bf16"},
        # Nothing divides: odd rows and columns, K not a multiple of 128.
        {"name": "gemm_odd", "op": "gemm", "m": 777, "n": 1001, "k": 1376, "dtype": "fp32"},
        # Prefill through the fused QKV projection.
        {"name": "gemm_prefill", "op": "gemm", "m": 2048, "n": 6144, "k": 4096, "dtype": "bf16"},
        # The largest square product of the GEMM benchmark's table.
        {"name": "gemm_large", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},
        # One decoded token between two blocks, layer-scale gate.
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "groups": 1,
         "gate": "channel", "alpha": 1.0, "dtype": "bf16"},
        # Odd rows of odd length, one gate value per row, scaled residual, fp16.
        {"name": "norm_odd", "op": "norm", "rows": 1001, "cols": 2047, "groups": 7,
         "gate": "row", "alpha": 0.81, "dtype": "fp16"},
        # A prefill batch of eight sequences, one gate row per sequence.
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "cols": 4096, "groups": 8,
         "gate": "group", "alpha": 1.0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(("quant", "gemm", "gemm", "norm"))
    if op == "quant":
        while True:
            rows, blocks = _log_int(rng, 1, 16384), _log_int(rng, 1, 896)
            if rows * blocks <= 14336 * 128:
                break
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        return {"op": op, "rows": rows, "cols": 32 * blocks,
                "pad": rng.choice((0, 0, 32 * blocks, rng.randrange(1, 100))), "dtype": dtype}
    if op == "gemm":
        while True:
            m, n, blocks = _log_int(rng, 1, 8192), _log_int(rng, 1, 28672), _log_int(rng, 1, 896)
            if rng.random() < 0.5:  # half of them at widths of whole tiles, as models have
                n, blocks = max(128, n // 128 * 128), max(4, blocks // 4 * 4)
            if m * n * blocks <= 8192 * 8192 * 256:
                break
        return {"op": op, "m": m, "n": n, "k": 32 * blocks,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    while True:
        groups, per, cols = _log_int(rng, 1, 64), _log_int(rng, 1, 4096), _log_int(rng, 1, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        if groups * per * cols <= 8192 * 4096:
            break
    return {"op": op, "rows": groups * per, "cols": cols, "groups": groups,
            "gate": rng.choice(("none", "channel", "row", "group", "full")),
            "alpha": rng.choice((1.0, round(rng.uniform(0.2, 3.0), 3))),
            "dtype": rng.choice(("bf16", "fp16", "fp32"))}


def work(case):
    if case["op"] == "quant":
        n, size = case["rows"] * case["cols"], SIZE[case["dtype"]]
        held = n // 2 + n // 32  # codes and scales: written by one call, read by the other
        return {"bytes": 2 * n * size + 2 * held, "flops": 4 * n}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k // 2 + k // 32) + m * n * SIZE[case["dtype"]],
                "flops": 2 * m * n * k}
    rows, cols, size = case["rows"], case["cols"], SIZE[case["dtype"]]
    gates = {"none": 0, "channel": cols, "row": rows, "group": case["groups"] * cols,
             "full": rows * cols}[case["gate"]]
    return {"bytes": (4 * rows * cols + 2 * cols + gates) * size, "flops": 10 * rows * cols}


# ---- inputs --------------------------------------------------------------------


def _random(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, cols):
    # Token magnitudes vary, and a few channels are far larger than the others.
    x = _random(gen, rows, cols) * torch.exp(0.5 * _random(gen, rows, 1))
    return x * torch.where(_random(gen, 1, cols) > 2.5, 12.0, 1.0)


def _held(values):
    """Codes [rows, cols / 2] (low nibble first) and scale bytes in tiles of 128
    rows x 4 blocks: byte (r % 32) * 16 + (r // 32) * 4 + block of a tile."""
    rows, cols = values.shape
    index, exponent = _encode(values)
    index = index.to(torch.uint8).reshape(rows, cols // 2, 2)
    codes = (index[..., 0] | (index[..., 1] << 4)).contiguous()
    tiles_m, tiles_k = -(-rows // 128), -(-cols // 128)
    flat = torch.zeros(tiles_m * 128, tiles_k * 4, dtype=torch.uint8, device=values.device)
    flat[:rows, :cols // 32] = exponent.to(torch.uint8)
    tiled = flat.reshape(tiles_m, 4, 32, tiles_k, 4).permute(0, 3, 2, 1, 4).contiguous()
    return codes, tiled.reshape(tiles_m, tiles_k, 512)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "quant":
        rows, cols = case["rows"], case["cols"]
        x = _activations(gen, rows, cols + case["pad"]).to(dtype)
        return {"case": case, "x": x[:, :cols]}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        a, a_scales = _held(_activations(gen, m, k))
        b, b_scales = _held(_random(gen, n, k) * k ** -0.5)
        return {"case": case, "a": a, "a_scales": a_scales, "b": b, "b_scales": b_scales}
    rows, cols, groups = case["rows"], case["cols"], case["groups"]
    per = rows // groups
    shape = {"none": None, "channel": (cols,), "row": (groups, per, 1),
             "group": (groups, 1, cols), "full": (groups, per, cols)}[case["gate"]]
    return {
        "case": case,
        "x": (3.0 * _random(gen, groups, per, cols)).to(dtype),
        "residual": _activations(gen, rows, cols).reshape(groups, per, cols).to(dtype),
        "post_weight": (1.0 + 0.2 * _random(gen, cols)).to(dtype),
        "pre_weight": (1.0 + 0.2 * _random(gen, cols)).to(dtype),
        "gate": None if shape is None else (0.5 * _random(gen, *shape)).to(dtype),
    }


# ---- plain forms -----------------------------------------------------------------


@functools.lru_cache(maxsize=8)
def _levels(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)


def _encode(x):
    """e2m1 codes (0..15) [rows, cols] and scale exponents (0..254) [rows, cols / 32]."""
    rows, cols = x.shape
    blocks = x.float().reshape(rows, cols // 32, 32)
    biased = blocks.abs().amax(dim=-1).view(torch.int32) >> 23  # floor(log2) + 127
    exponent = (biased - 2).clamp(min=0)
    v = blocks * ((254 - exponent) << 23).view(torch.float32).unsqueeze(-1)
    mag = v.abs()
    index = ((mag > 0.25).int() + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75) + (mag > 2.5)
             + (mag >= 3.5) + (mag > 5.0))
    index = torch.where(v < 0, index + 8, index)
    return index.reshape(rows, cols), exponent


def _power(exponent):
    """2^(exponent - 127) as fp32; the smallest is subnormal."""
    bits = exponent.int() << 23
    return torch.where(bits == 0, torch.full_like(bits, 1 << 22), bits).view(torch.float32)


def _decode(codes, tiled):
    rows, cols = codes.shape[0], 2 * codes.shape[1]
    index = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(rows, cols)
    levels = _levels(codes.device)
    table = torch.cat((levels, -levels))
    tiles_m, tiles_k = tiled.shape[:2]
    flat = tiled.reshape(tiles_m, tiles_k, 32, 4, 4).permute(0, 3, 2, 1, 4)
    scales = _power(flat.reshape(tiles_m * 128, tiles_k * 4)[:rows, :cols // 32])
    return table[index.int()].reshape(rows, cols // 32, 32).mul_(scales.unsqueeze(-1)).reshape(rows, cols)


def _rms(v):
    return v * torch.rsqrt(v.square().mean(dim=-1, keepdim=True) + EPS)


def run(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "quant":
        x = state["x"]
        if own:
            codes, scales = _api().mxfp4_quantize(x)
            return _api().mxfp4_dequantize(codes, scales, dtype)
        index, exponent = _encode(x)
        q = _levels(x.device)[index & 7]
        q = torch.where(index >= 8, -q, q).reshape(x.shape[0], -1, 32)
        return (q * _power(exponent).unsqueeze(-1)).reshape(x.shape).to(dtype)
    if case["op"] == "gemm":
        if own:
            return _api().mxfp4_gemm(state["a"], state["a_scales"], state["b"], state["b_scales"],
                                     out_dtype=dtype)
        a, b = _decode(state["a"], state["a_scales"]), _decode(state["b"], state["b_scales"])
        return (a @ b.t()).to(dtype)
    x, residual, gate = state["x"], state["residual"], state["gate"]
    if own:
        return _api().sandwich_rmsnorm(x, residual, state["post_weight"], state["pre_weight"], EPS,
                                       gate=gate, residual_scale=case["alpha"])
    branch = _rms(x.float()) * state["post_weight"].float()
    if gate is not None:
        branch = branch * gate.float()
    h = case["alpha"] * residual.float() + branch
    return (_rms(h) * state["pre_weight"].float()).to(dtype), h.to(dtype)


# ---- the definitions in 64 bits -----------------------------------------------------


def _two_to(n):
    """2^n in fp64 from its bits: pow() on a GPU may be off by an ulp, which moves ties."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _values64(codes, tiled):
    rows, cols = codes.shape[0], 2 * codes.shape[1]
    nibbles = torch.empty(rows, cols, dtype=torch.int32, device=codes.device)
    nibbles[:, 0::2] = codes % 16
    nibbles[:, 1::2] = codes // 16
    low = nibbles % 8
    two, one = low // 2, low % 2  # exponent and mantissa bits of e2m1, bias 1
    mag = torch.where(two == 0, 0.5 * one.double(), (1 + 0.5 * one.double()) * _two_to(two - 1))
    r = torch.arange(rows, device=codes.device).unsqueeze(1)
    j = torch.arange(cols // 32, device=codes.device).unsqueeze(0)
    byte = tiled[r // 128, j // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4]
    scale = _two_to(byte.int() - 127)
    signed = torch.where(nibbles >= 8, -mag, mag)
    return signed * scale.repeat_interleave(32, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quant":
        x = state["x"].double()
        blocks = x.reshape(x.shape[0], -1, 32)
        top = blocks.abs().max(dim=-1, keepdim=True).values
        e = torch.frexp(top).exponent - 3  # top = m * 2^exponent, m in [.5, 1)
        scale = _two_to(e.clamp(min=-127))
        v = (blocks / scale).abs().clamp(max=6.0)
        # The spacing of e2m1: .5 below 2, 1 up to 4, 2 above; round() takes ties to even.
        step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0)).double()
        q = torch.round(v / step) * step
        return (torch.sign(blocks) * q * scale).reshape(x.shape)
    if case["op"] == "gemm":
        a = _values64(state["a"], state["a_scales"])
        return a @ _values64(state["b"], state["b_scales"]).t()
    x, residual = state["x"].double(), state["residual"].double()
    branch = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["cols"] + EPS)
    branch = branch * state["post_weight"].double()
    if state["gate"] is not None:
        branch = branch * state["gate"].double()
    h = case["alpha"] * residual + branch
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["cols"] + EPS)
    return y * state["pre_weight"].double(), h
