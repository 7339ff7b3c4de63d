"""What is measured of the FP8 dense path: projections whose weights and activations are 8-bit floats.

Values are held as e4m3 codes with an FP32 scale for each block of 128: activations per row and 128
columns, weights per 128 x 128. Activations are quantised (``quantize``), on their own or behind the
residual add and RMSNorm (``norm``), and multiplied by the weights (``matmul``); a gated feed-forward
block (``ffn``) multiplies by gate and up weights, applies the activation, quantises the product and
multiplies by the down weights.

With ``own`` false, ``run`` computes each operator in its plain form (elementary torch operations in
32 bits, rounded once at the end); with ``own`` true it calls ``qk_b200``.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_BLOCK = 128
_MOST = 448.0          # the largest e4m3 value
_LEAST = 2.0 ** -100   # the smallest maximum of a block that counts


def listed():
    return [
        # the attention outputs of a decode step of 64 sequences: latency
        dict(name="quantize b64", op="quantize", rows=64, width=4096, dtype="bf16"),
        # a long prompt's activations
        dict(name="quantize prompt 32768", op="quantize", rows=32768, width=4096, dtype="bf16"),
        # FP32 values, a width that no block divides
        dict(name="quantize odd 8111", op="quantize", rows=8111, width=1111, dtype="f32"),
        # the norm before the projections in a decode step of 8 sequences
        dict(name="norm b8", op="norm", rows=8, width=2048, residual=True),
        # the same over a prompt chunk
        dict(name="norm prompt 16384", op="norm", rows=16384, width=2048, residual=True),
        # q, gate, k and v of one sequence's new token: latency and the weights' bytes
        dict(name="matmul b1 qkv", op="matmul", rows=1, k=2048, n=9216, x="bf16", out="bf16"),
        # the output projection of 64 sequences
        dict(name="matmul b64 out", op="matmul", rows=64, k=4096, n=2048, x="bf16", out="bf16"),
        # odd sizes throughout, FP32 results
        dict(name="matmul odd 333", op="matmul", rows=333, k=1111, n=1000, x="bf16", out="f32"),
        # a prompt chunk behind the norm: activations that are FP8 already
        dict(name="matmul prompt 16384", op="matmul", rows=16384, k=2048, n=9216, x="fp8", out="bf16"),
        # a shared expert's block for 4 sequences
        dict(name="ffn b4", op="ffn", rows=4, k=2048, inner=512),
        # a dense layer's block for 32 sequences
        dict(name="ffn b32", op="ffn", rows=32, k=2048, inner=6144),
        # and for a prompt chunk
        dict(name="ffn prompt 8192", op="ffn", rows=8192, k=2048, inner=6144),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "matmul", "matmul", "matmul", "ffn", "ffn"])
    rows = _log_int(rng, 1, 16384)
    if op == "quantize":
        return dict(op=op, rows=rows, width=_log_int(rng, 64, 8192), dtype=rng.choice(["bf16", "f32"]))
    if op == "norm":
        return dict(op=op, rows=rows, width=8 * _log_int(rng, 16, 1024), residual=rng.random() < 0.7)

    def side(low, high):  # whole blocks, or anything
        return _BLOCK * _log_int(rng, low, high) if rng.random() < 0.6 else _log_int(rng, low * _BLOCK, high * _BLOCK)

    if op == "matmul":
        k, n = side(2, 64), side(1, 96)
        while rows * k * n > 16384 * 2048 * 9216:
            rows = rows * 2 // 3
        return dict(op=op, rows=rows, k=k, n=n, x=rng.choice(["bf16", "fp8"]), out=rng.choice(["bf16", "bf16", "f32"]))
    k, inner = side(2, 32), side(2, 48)
    while rows * k * inner > 8192 * 2048 * 6144:
        rows = rows * 2 // 3
    return dict(op=op, rows=rows, k=k, inner=inner)


# ---- inputs ------------------------------------------------------------------------------


def _device():
    return torch.device("cuda")


def _activations(g, rows, width, dtype):
    """Rows of unequal size with a few channels that are much larger than the others."""
    x = torch.randn((rows, width), generator=g, device=g.device)
    x *= torch.exp(torch.randn((rows, 1), generator=g, device=g.device) * 0.5)
    x *= torch.exp(torch.randn((1, width), generator=g, device=g.device) * 0.7)
    return x.to(dtype)


def _pitched(codes):
    """Rows of codes that begin on 16 bytes, as a program lays out its weights once."""
    rows, width = codes.shape
    store = torch.zeros((rows, (width + 15) // 16 * 16), dtype=torch.uint8, device=codes.device)
    store[:, :width] = codes.view(torch.uint8)
    return store.view(torch.float8_e4m3fn)[:, :width]


def _weights(g, n, k):
    """e4m3 codes [n, k] and scales [blocks of n, blocks of k] of N(0, 0.02) weights."""
    w = torch.randn((n, k), generator=g, device=g.device) * 0.02
    rows, columns = (n + _BLOCK - 1) // _BLOCK, (k + _BLOCK - 1) // _BLOCK
    full = torch.zeros((rows * _BLOCK, columns * _BLOCK), device=g.device)
    full[:n, :k] = w
    most = full.view(rows, _BLOCK, columns, _BLOCK).abs().amax((1, 3)).clamp(min=_LEAST)
    by = (_MOST / most).repeat_interleave(_BLOCK, 0).repeat_interleave(_BLOCK, 1)[:n, :k]
    return _pitched((w * by).to(torch.float8_e4m3fn)), most / _MOST


def prepare(case, seed):
    g = torch.Generator(device=_device()).manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        x = _activations(g, case["rows"], case["width"], dtype)
        x[-1, :_BLOCK] = 0  # a block of zeros
        return dict(op=op, x=x)
    if op == "norm":
        x = _activations(g, case["rows"], case["width"], torch.bfloat16)
        y = _activations(g, case["rows"], case["width"], torch.bfloat16) if case["residual"] else None
        gamma = (1 + 0.2 * torch.randn(case["width"], generator=g, device=g.device)).to(torch.bfloat16)
        return dict(op=op, x=x, residual=y, gamma=gamma, eps=1e-6)
    x = _activations(g, case["rows"], case["k"], torch.bfloat16)
    if op == "matmul":
        s = dict(op=op, weights=_weights(g, case["n"], case["k"]),
                 out=torch.bfloat16 if case["out"] == "bf16" else torch.float32)
        if case["x"] == "bf16":
            return dict(s, x=x)
        codes, scales = _quantized(x.float())
        return dict(s, codes=_pitched(codes), scales=scales)
    # small enough that products, not the activation's tails, decide
    return dict(op=op, x=x * 0.25, gate=_weights(g, case["inner"], case["k"]), up=_weights(g, case["inner"], case["k"]),
                down=_weights(g, case["k"], case["inner"]))


# ---- the framework's operators -------------------------------------------------------------


def _run_own(s):
    folder = str(Path(__file__).resolve().parents[1] / "data-synth-tpu_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from qk_b200.fp8 import Fp8Rows, Fp8Weights, fp8_matmul, gated_ffn_fp8, quantize_fp8, rms_norm_fp8

    if s["op"] == "quantize":
        return list(quantize_fp8(s["x"]))
    if s["op"] == "norm":
        rows, total = rms_norm_fp8(s["x"], s["gamma"], s["eps"], residual=s["residual"])
        return [rows.codes, rows.scales] + ([] if total is None else [total])
    if s["op"] == "matmul":
        x = s["x"] if "x" in s else Fp8Rows(s["codes"], s["scales"])
        return fp8_matmul(x, Fp8Weights(*s["weights"]), output_dtype=s["out"])
    return gated_ffn_fp8(s["x"], Fp8Weights(*s["gate"]), Fp8Weights(*s["up"]), Fp8Weights(*s["down"]))


# ---- the plain forms -----------------------------------------------------------------------


def _quantized(x):
    """Codes [rows, width] and scales [blocks, rows] of FP32 values."""
    rows, width = x.shape
    blocks = (width + _BLOCK - 1) // _BLOCK
    full = x if width == blocks * _BLOCK else torch.cat([x, x.new_zeros((rows, blocks * _BLOCK - width))], 1)
    full = full.view(rows, blocks, _BLOCK)
    most = full.abs().amax(2).clamp(min=_LEAST)
    # one division: a product with a rounded reciprocal would leave the ties, frequent in BF16, to chance
    codes = (full * _MOST / most[:, :, None]).to(torch.float8_e4m3fn)
    return codes.view(rows, -1)[:, :width], (most / _MOST).t().contiguous()


def _values(codes, scales):
    """The FP32 values of codes with a scale for every row and block."""
    by = scales.repeat_interleave(_BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * by


def _weight_values(weights):
    codes, scales = weights
    return _values(codes, scales.repeat_interleave(_BLOCK, 0)[:codes.shape[0]])


def _plain(s):
    if s["op"] == "quantize":
        return list(_quantized(s["x"].float()))
    if s["op"] == "norm":
        x, total = s["x"], None
        if s["residual"] is not None:
            x = total = (x.float() + s["residual"].float()).to(torch.bfloat16)
        x = x.float()
        by = torch.rsqrt((x * x).mean(1) + s["eps"])
        # the row's factor moves no code: it goes into the scales
        codes, scales = _quantized(x * s["gamma"].float())
        return [codes, scales * by] + ([] if total is None else [total])
    codes, scales = _quantized(s["x"].float()) if "x" in s else (s["codes"], s["scales"])
    x = _values(codes, scales.t())
    if s["op"] == "matmul":
        return torch.matmul(x, _weight_values(s["weights"]).t()).to(s["out"])
    gate = torch.matmul(x, _weight_values(s["gate"]).t())
    up = torch.matmul(x, _weight_values(s["up"]).t())
    codes, scales = _quantized(gate / (1 + torch.exp(-gate)) * up)
    return torch.matmul(_values(codes, scales.t()), _weight_values(s["down"]).t()).to(torch.bfloat16)


def run(state):
    return _run_own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------


def _blocks(n):
    return (n + _BLOCK - 1) // _BLOCK


def work(case):
    op, rows = case["op"], case["rows"]
    if op in ("quantize", "norm"):
        width = case["width"]
        size = 4 if case.get("dtype") == "f32" else 2
        more = 2 * rows * width * 2 if case.get("residual") else 0  # the other addend in, the sum out
        return {"bytes": rows * (width * (size + 1) + 4 * _blocks(width)) + more + (2 * width if op == "norm" else 0),
                "flops": (3 if op == "quantize" else 7) * rows * width}

    def weights(n, k):
        return n * k + 4 * _blocks(n) * _blocks(k)

    k = case["k"]
    if op == "matmul":
        n = case["n"]
        x = rows * k * 2 if case["x"] == "bf16" else rows * (k + 4 * _blocks(k))
        return {"bytes": x + weights(n, k) + rows * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * rows * n * k}
    inner = case["inner"]
    return {"bytes": 2 * rows * k * 2 + 2 * weights(inner, k) + weights(k, inner), "flops": 6 * rows * k * inner}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def _e4m3(x):
    """The nearest values of 4 bits of exponent and 3 of fraction, ties to even."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_rows(x):
    rows, width = x.shape
    codes = torch.empty_like(x)
    scales = x.new_empty((_blocks(width), rows))
    for b in range(_blocks(width)):
        part = x[:, b * _BLOCK:(b + 1) * _BLOCK]
        most = part.abs().amax(1).clamp(min=_LEAST)
        scales[b] = most / _MOST
        codes[:, b * _BLOCK:(b + 1) * _BLOCK] = _e4m3(part * _MOST / most[:, None])
    return codes, scales


def _exact_product(codes, scales, weights):
    out = 0
    wc, ws = weights[0].double(), weights[1].double()
    for b in range(scales.shape[0]):
        at = slice(b * _BLOCK, (b + 1) * _BLOCK)
        by = ws[torch.arange(wc.shape[0], device=wc.device) // _BLOCK, b]
        out = out + (codes[:, at] @ wc[:, at].t()) * scales[b][:, None] * by
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        return list(_exact_rows(s["x"].double()))
    if s["op"] == "norm":
        x = s["x"].double()
        total = None
        if s["residual"] is not None:
            total = x + s["residual"].double()
            x = total.to(torch.bfloat16).double()  # what is normed is the sum that is kept
        codes, scales = _exact_rows(x * s["gamma"].double())
        return [codes, scales / torch.sqrt((x ** 2).sum(1) / x.shape[1] + s["eps"])] + ([] if total is None else [total])
    codes, scales = _exact_rows(s["x"].double()) if "x" in s else (s["codes"].double(), s["scales"].double())
    if s["op"] == "matmul":
        return _exact_product(codes, scales, s["weights"])
    gate, up = (_exact_product(codes, scales, s[name]) for name in ("gate", "up"))
    return _exact_product(*_exact_rows(gate * torch.sigmoid(gate) * up), s["down"])
