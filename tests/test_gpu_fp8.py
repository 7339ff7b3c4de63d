"""FP8 dense path on the GPU against its definition in 64 bits (plain NumPy): e4m3 codes with an FP32
scale per block of 128, the residual norm that leaves as codes, the products and the gated block.

Tolerances. Codes are compared exactly where the quotient 448 x / m cannot lie near a border without
being one: x and m have at most 16 significant bits (BF16, or a product of two), so a quotient that is
no border is at least 2^-21 of its size from the next, and FP32 decides as 64 bits do. Sums of FP32
products are off by at most one unit of 2^-23 of the terms' magnitudes per addition: 128 within a block
(the products of codes are exact) and one per block. Outputs are rounded by half a step on top.
"""

import numpy as np
import pytest

from util import to_f32

pytestmark = pytest.mark.gpu

BLOCK = 128
LEAST = 2.0 ** -100


def blocks(n):
    return -(-n // BLOCK)


def e4m3(x):
    """The nearest e4m3 values, ties to even."""
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(x / step) * step


def row_most(x):
    full = np.zeros((x.shape[0], blocks(x.shape[1]) * BLOCK))
    full[:, :x.shape[1]] = np.abs(x)
    return np.maximum(full.reshape(x.shape[0], -1, BLOCK).max(2), LEAST)


def spread(a, width):
    """A value per block -> one per column."""
    return np.repeat(a, BLOCK, axis=-1)[..., :width]


def quantized(x):
    most = row_most(x)
    return e4m3(x * 448 / spread(most, x.shape[1])), most / 448


def values(rows):
    """The 64-bit values of Fp8Rows, and the codes alone."""
    codes = to_f32(rows.codes).astype(np.float64)
    return codes * spread(to_f32(rows.scales).astype(np.float64).T, codes.shape[1]), codes


def weight_values(w):
    codes = to_f32(w.codes).astype(np.float64)
    scales = spread(to_f32(w.scales).astype(np.float64), codes.shape[1])
    return codes * np.repeat(scales, BLOCK, axis=0)[:codes.shape[0]]


def activations(rows, width, device, seed=0, dtype=None):
    import torch

    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn((rows, width), generator=g, device=device)
    x *= torch.exp(torch.randn((rows, 1), generator=g, device=device))
    return x.to(dtype or torch.bfloat16)


def packed(n, k, device, seed=1):
    from qk_b200.fp8 import pack_fp8

    return pack_fp8(activations(n, k, device, seed) * 0.05)


def sum_error(x, w):
    return (BLOCK + blocks(x.shape[1])) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def check_product(got, x, w, half_step):
    want, room = x @ w.T, sum_error(x, w)
    off = np.abs(to_f32(got).astype(np.float64) - want)
    assert np.all(off <= half_step * (np.abs(want) + room) + room + 1e-38), float(np.max(off / (np.abs(want) + room + 1e-38)))


# ---- quantisation -----------------------------------------------------------------------------


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 127), (5, 129), (64, 2048), (37, 4104), (300, 1111), (2, 40000)])
def test_rows_are_quantised_by_the_rule(cuda_device, rows, width):
    from qk_b200.fp8 import quantize_fp8

    x = activations(rows, width, cuda_device, rows + width)
    x[-1, :BLOCK] = 0
    got = quantize_fp8(x)
    codes, scales = quantized(to_f32(x).astype(np.float64))
    assert got.codes.shape == x.shape and got.scales.shape == (blocks(width), rows)
    assert np.array_equal(to_f32(got.codes), codes.astype(np.float32))
    assert np.array_equal(to_f32(got.scales), scales.T.astype(np.float32))


@pytest.mark.parametrize("rows,width", [(64, 2048), (33, 1111)])
def test_fp32_rows(cuda_device, rows, width):
    """24 bits can lie as near to a border as FP32 can tell: there either neighbour will do."""
    import torch

    from qk_b200.fp8 import quantize_fp8

    x = activations(rows, width, cuda_device, 3, torch.float32)
    got = quantize_fp8(x)
    x = to_f32(x).astype(np.float64)
    quotient = x * 448 / spread(row_most(x), width)
    codes = to_f32(got.codes)
    near = np.abs(e4m3(quotient * (1 + 2.0 ** -21)) - e4m3(quotient * (1 - 2.0 ** -21))) > 0
    assert np.all((codes == e4m3(quotient)) | near) and near.mean() < 1e-3
    assert np.array_equal(to_f32(got.scales), (row_most(x) / 448).T.astype(np.float32))


def test_ties_go_to_even(cuda_device):
    """A maximum of 448 makes every short value its own quotient: all borders between codes, exactly."""
    import torch

    from qk_b200.fp8 import quantize_fp8

    bits = np.arange(1, 0x7e, dtype=np.uint8)
    grid = torch.from_numpy(bits).view(torch.float8_e4m3fn).float().numpy()
    border = (grid[1:] + grid[:-1]) / 2
    for most in (448.0, 448.0 * 1.25, 448.0 * 1.625 * 2 ** -20):
        x = np.zeros((1, 128), np.float32)
        x[0, :len(border)] = border * (most / 448)
        x[0, 127] = most
        want = quantized(x.astype(np.float64))[0].astype(np.float32)
        xt = torch.from_numpy(x).to(cuda_device)
        assert np.array_equal(to_f32(quantize_fp8(xt).codes), want)
        if torch.equal(xt.to(torch.bfloat16).float(), xt):  # 13 / 8 times a border has a bit too many
            assert np.array_equal(to_f32(quantize_fp8(xt.to(torch.bfloat16)).codes), want)
        else:
            assert most < 1


def test_strided_and_shifted_rows(cuda_device):
    import torch

    from qk_b200.fp8 import quantize_fp8

    wide = activations(20, 1000, cuda_device, 5)
    for view in (wide[:, 8:520], wide[:, 3:700], wide[::3], wide[:, ::2], wide.t(), wide[:0]):
        got, want = quantize_fp8(view), quantize_fp8(view.clone(memory_format=torch.contiguous_format))
        assert torch.equal(got.codes.float(), want.codes.float()) and torch.equal(got.scales, want.scales)


def test_extreme_blocks(cuda_device):
    import torch

    from qk_b200.fp8 import quantize_fp8

    x = torch.ones((6, 256), device=cuda_device)
    x[0, 3] = float("inf")
    x[1, 5] = float("nan")
    x[2] = 3e38          # near FP32's end
    x[3] = 2.0 ** -126   # far below what counts
    x[4, :128] = 0
    x[5, 7] = -float("inf")
    got = quantize_fp8(x)
    codes, scales = got.codes.float(), got.scales
    value = codes * scales.t().repeat_interleave(128, 1)
    assert not torch.isfinite(value[0, :128]).any() and not torch.isfinite(value[5, :128]).any()
    assert torch.isnan(value[1, :128]).all()
    assert (codes[2] == 448).all() and torch.isfinite(value[2]).all()
    assert (value[3] == 0).all() and (value[4, :128] == 0).all()
    assert (value[[0, 1, 4, 5], 128:] == 1).all()  # their other blocks


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (127, 130), (300, 1111), (9216, 2048)])
def test_weights_are_quantised_by_blocks(cuda_device, n, k):
    from qk_b200.fp8 import pack_fp8

    w = activations(n, k, cuda_device, n)
    got = pack_fp8(w)
    w = to_f32(w).astype(np.float64)
    full = np.zeros((blocks(n) * BLOCK, blocks(k) * BLOCK))
    full[:n, :k] = np.abs(w)
    most = np.maximum(full.reshape(blocks(n), BLOCK, blocks(k), BLOCK).max((1, 3)), LEAST)
    by = np.repeat(spread(most, k), BLOCK, axis=0)[:n]
    assert np.array_equal(to_f32(got.codes), e4m3(w * 448 / by).astype(np.float32))
    assert np.array_equal(to_f32(got.scales), (most / 448).astype(np.float32))


# ---- norm -------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,width", [(1, 8), (3, 136), (8, 2048), (5, 8192), (700, 2048), (257, 1000)])
@pytest.mark.parametrize("add", [False, True])
def test_norm_leaves_as_codes(cuda_device, rows, width, add):
    import torch

    from qk_b200.fp8 import rms_norm_fp8

    x = activations(rows, width, cuda_device, 1)
    y = activations(rows, width, cuda_device, 2) if add else None
    gamma = (1 + 0.3 * torch.randn(width, device=cuda_device)).to(torch.bfloat16)
    x[-1] = 0
    if add:
        y[-1] = 0
    got, total = rms_norm_fp8(x, gamma, 1e-5, residual=y)
    if add:
        assert torch.equal(total, (x.float() + y.float()).to(torch.bfloat16))
        x = total
    else:
        assert total is None
    x, gamma = to_f32(x).astype(np.float64), to_f32(gamma).astype(np.float64)
    codes, scales = quantized(x * gamma)
    assert np.array_equal(to_f32(got.codes), codes.astype(np.float32))
    scales = (scales / np.sqrt((x ** 2).mean(1) + 1e-5)[:, None]).T
    # the sum of squares: at most 45 additions one behind another, the mean, the root, two products
    assert np.all(np.abs(to_f32(got.scales) - scales) <= 2.0 ** -18 * scales)


# ---- products ---------------------------------------------------------------------------------


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 128, 128), (1, 2048, 9216), (3, 100, 7), (8, 4096, 2048), (16, 2048, 300),
                                   (31, 1111, 1000), (64, 4096, 2048), (65, 640, 520), (128, 16384, 256), (129, 257, 255),
                                   (200, 384, 136), (333, 1111, 1000), (1000, 2048, 2304),
                                   # more tiles than SMs: a CTA has all of K, more blocks than it can quantise
                                   (1, 8192, 19000), (2, 16384, 19100), (40, 2176, 19000)])
@pytest.mark.parametrize("f32", [False, True])
def test_matmul(cuda_device, m, k, n, f32):
    import torch

    from qk_b200.fp8 import check_status, fp8_matmul, quantize_fp8

    x, w = activations(m, k, cuda_device, m), packed(n, k, cuda_device)
    dtype = torch.float32 if f32 else torch.bfloat16
    got = fp8_matmul(x, w, output_dtype=dtype)
    again = fp8_matmul(quantize_fp8(x), w, output_dtype=dtype)
    check_status(cuda_device)
    assert torch.equal(got, again) and got.dtype == dtype and got.shape == (m, n)
    check_product(got, values(quantize_fp8(x))[0], weight_values(w), 2.0 ** -24 if f32 else 2.0 ** -8)


@pytest.mark.parametrize("m,k,inner", [(1, 2048, 512), (4, 128, 128), (16, 300, 200), (33, 1111, 100), (64, 2048, 512),
                                       (100, 512, 1000), (129, 256, 257), (300, 2048, 640)])
def test_gated(cuda_device, m, k, inner):
    import torch

    from qk_b200.fp8 import check_status, fp8_matmul, gated_ffn_fp8, gated_fp8, quantize_fp8

    x, gate, up = activations(m, k, cuda_device, m) * 0.5, packed(inner, k, cuda_device, 2), packed(inner, k, cuda_device, 3)
    down = packed(192, inner, cuda_device, 4)
    got = gated_fp8(x, gate, up)
    xv, gv, uv = values(quantize_fp8(x))[0], weight_values(gate), weight_values(up)
    g, u = xv @ gv.T, xv @ uv.T
    silu = g / (1 + np.exp(-g))
    h = silu * u
    # |silu'| stays below 1.1; exponential and quotient within 2^-16
    error = 1.1 * np.abs(u) * sum_error(xv, gv) + np.abs(silu) * sum_error(xv, uv) + 2.0 ** -16 * np.abs(h)
    most = row_most(h)
    worst = np.array([[error[r, b * BLOCK:(b + 1) * BLOCK].max() for b in range(blocks(inner))] for r in range(m)])
    assert np.all(np.abs(to_f32(got.scales).T - most / 448) <= (worst + 2.0 ** -22 * most) / 448)
    value, codes = values(got)
    _, e = np.frexp(codes)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3) * spread(to_f32(got.scales).astype(np.float64).T, inner)
    assert np.all(np.abs(value - h) <= step / 2 * (1 + 2.0 ** -20) + 2 * error)
    out = gated_ffn_fp8(x, gate, up, down)
    assert torch.equal(out, fp8_matmul(got, down))
    check_status(cuda_device)
    check_product(out, value, weight_values(down), 2.0 ** -8)


# More rows: tiles of 256 x 128, with a ragged end on every side, and in several rounds; of 256 x 256 in one round and
# in two; of few rows after all, 128 at a time.
@pytest.mark.parametrize("m,k,n", [(65, 256, 512), (129, 130, 777), (300, 384, 130), (700, 1000, 3001), (1500, 520, 5000), (257, 2048, 9216),
                                   (512, 2000, 9216), (520, 2040, 9100), (256, 4096, 2048), (250, 8100, 2041), (390, 500, 12200),
                                   # as much shared memory as a CTA can have
                                   (70, 8192, 3840), (66, 8100, 3777)])
@pytest.mark.parametrize("f32", [False, True])
def test_matmul_of_more_rows(cuda_device, m, k, n, f32):
    test_matmul(cuda_device, m, k, n, f32)


@pytest.mark.parametrize("m,k,inner", [(40, 2048, 512), (33, 600, 6000), (500, 4100, 760), (513, 300, 3001), (1000, 256, 1000),
                                       (900, 2048, 5000)])
def test_gated_of_more_rows(cuda_device, m, k, inner):
    test_gated(cuda_device, m, k, inner)


# ---- together, and as the decoder uses them ----------------------------------------------------


def test_a_layer_of_fp8_operators_matches_its_parts(cuda_device):
    """Norm, projection, residual norm and feed-forward one behind another, as a dense layer runs them:
    each operator's output is checked against 64 bits from the operator's own input."""
    import torch

    from qk_b200.fp8 import check_status, fp8_matmul, gated_ffn_fp8, gated_fp8, rms_norm_fp8

    rows, hidden, inner = 24, 512, 640
    x = activations(rows, hidden, cuda_device, 7)
    gamma = (1 + 0.1 * torch.randn(hidden, device=cuda_device)).to(torch.bfloat16)
    w, gate, up = packed(hidden, hidden, cuda_device), packed(inner, hidden, cuda_device, 2), packed(inner, hidden, cuda_device, 3)
    down = packed(hidden, inner, cuda_device, 4)
    h, _ = rms_norm_fp8(x, gamma)
    y = fp8_matmul(h, w)
    check_product(y, values(h)[0], weight_values(w), 2.0 ** -8)
    h, x1 = rms_norm_fp8(x, gamma, residual=y)
    assert torch.equal(x1, (x.float() + y.float()).to(torch.bfloat16))
    out = gated_ffn_fp8(h, gate, up, down)
    check_product(out, values(gated_fp8(h, gate, up))[0], weight_values(down), 2.0 ** -8)
    check_status(cuda_device)


def decoder_of(device, dense):
    from qk_b200.decoder import StackConfig, SyntheticDecoder

    return SyntheticDecoder(StackConfig(layers=2, experts=16, top_k=2, qtype="Q4_K", context=96, dense=dense), device, seed=5)


@pytest.mark.parametrize("batch", [1, 3, 40])
def test_decode_step_with_fp8_projections(cuda_device, batch):
    """The step's projections are the products of its own inputs, and a captured step gives the eager one's bits."""
    import torch

    model = decoder_of(cuda_device, "fp8")
    state = model.state(batch, seed=2)
    x0 = state.x.clone()
    state.step()
    eager = state.x.clone()
    L = model.layers[-1]
    codes = to_f32(state.fp8.codes).astype(np.float64)
    h = codes * spread(to_f32(state.fp8.scales).astype(np.float64).T, codes.shape[1])
    check_product(state.qkv, h, weight_values(L.w_qkv), 2.0 ** -8)
    o = to_f32(state.o).reshape(batch, -1).astype(np.float64)
    oc, os = quantized(o)
    check_product(state.a, oc * spread(os.astype(np.float32).astype(np.float64), o.shape[1]), weight_values(L.w_o), 2.0 ** -8)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(cuda_device)
    with torch.cuda.graph(graph):
        state.step()
    state.x.copy_(x0)
    graph.replay()
    torch.cuda.synchronize(cuda_device)
    assert torch.equal(state.x.view(torch.int16), eager.view(torch.int16))


def test_prefill_with_fp8_projections_matches_steps(cuda_device):
    """As for BF16 projections: one pass over the prompt and token by token agree."""
    import torch

    from qk_b200.generate import StaticGeneration

    model = decoder_of(cuda_device, "fp8")
    batch, prompt = 3, 64
    gen = StaticGeneration(model, batch, prompt, 8, vocab=1000, seed=1)
    gen.prefill()
    ref = StaticGeneration(model, batch, prompt, 8, vocab=1000, seed=1)
    for t in range(prompt):
        ref.state.x.copy_(ref.embedding.index_select(0, ref.prompt_ids[:, t]))
        ref.state.positions.fill_(t)
        ref.state.step()
    ref._choose(0)
    torch.cuda.synchronize(cuda_device)
    a, b = to_f32(gen.logits), to_f32(ref.logits)
    # a code of 4 bits may go the other way for a last bit of its input: twice the room of BF16 projections
    assert np.abs(a - b).max() < 0.1 * np.abs(b).max()
    out = gen.decode().cpu().numpy()
    assert out.min() >= 0 and out.max() < 1000 and int(gen.nonfinite.item()) == 0
    gen.close()
    ref.close()


def test_speculative_generation_with_fp8_projections(cuda_device):
    from qk_b200.speculate import SpeculativeGeneration

    model = decoder_of(cuda_device, "fp8")
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 600, n).tolist() for n in (5, 17)]
    gen = SpeculativeGeneration(model, 2, 64, nodes=4, page_size=16, vocab=600)
    gen.prefill(prompts)
    rows = gen.generate(6)
    for row, prompt in zip(rows, prompts):
        assert row[:len(prompt)] == prompt and len(row) > len(prompt) + 5 and all(0 <= t < 600 for t in row)


def test_products_of_many_sizes(cuda_device):
    """Sizes at random: every number of tokens, splits of K and buffers, both forms."""
    import random

    import torch

    from qk_b200.fp8 import check_status, fp8_matmul, gated_ffn_fp8, gated_fp8, quantize_fp8

    rng = random.Random(11)
    for i in range(60):
        m = rng.choice([1, 2, 5, 9, 16, 17, 30, 33, 64, 65, 100, 128, 129, 260])
        k = rng.choice([16, 128, 8 * rng.randint(1, 700), rng.randint(1, 3000)])
        n = rng.choice([rng.randint(1, 600), 128 * rng.randint(1, 40), 9216])
        x, w = activations(m, k, cuda_device, i), packed(n, k, cuda_device, i)
        rows = quantize_fp8(x)
        got = fp8_matmul(x, w)
        assert torch.equal(got, fp8_matmul(rows, w)), (m, k, n)
        check_product(got, values(rows)[0], weight_values(w), 2.0 ** -8)
        if n * k < 1 << 20:
            down = packed(rng.randint(1, 300), n, cuda_device, i)
            out = gated_ffn_fp8(x, w, w, down)
            assert torch.equal(out, fp8_matmul(gated_fp8(rows, w, w), down)), (m, k, n)
    check_status(cuda_device)


# ---- refusals, layouts, streams, graphs -----------------------------------------------------------


def test_mismatched_operands_are_refused(cuda_device):
    import torch

    from qk_b200.fp8 import Fp8Rows, Fp8Weights, fp8_matmul, fp8_weights, gated_ffn_fp8, quantize_fp8, rms_norm_fp8

    x, w = activations(3, 256, cuda_device), packed(128, 256, cuda_device)
    rows = quantize_fp8(x)
    with pytest.raises(ValueError):
        fp8_matmul(x[:, :128], w)
    with pytest.raises(ValueError):
        fp8_matmul(x, Fp8Weights(w.codes, w.scales.t()))
    with pytest.raises(ValueError):
        fp8_matmul(x, Fp8Weights(w.codes.cpu(), w.scales))
    with pytest.raises(ValueError):
        fp8_matmul(Fp8Rows(rows.codes, rows.scales.t()), w)
    with pytest.raises(ValueError):
        fp8_matmul(x, w, out=torch.empty((3, 128), device=cuda_device), output_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp8_matmul(x, w, out=torch.empty((128, 3), dtype=torch.bfloat16, device=cuda_device).t())
    with pytest.raises(ValueError):
        gated_ffn_fp8(x, w, packed(120, 256, cuda_device), w)
    with pytest.raises(ValueError):
        gated_ffn_fp8(x, w, w, w)
    with pytest.raises(ValueError):
        rms_norm_fp8(x, x[0].clone(), residual=x[:2])
    with pytest.raises(ValueError):
        fp8_weights(w.codes, w.scales[:, :1])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_outputs_over_their_inputs(m, cuda_device):
    """A product refuses an ``out`` that shares memory with ``x``; a feed-forward block may write over it."""
    import torch

    from qk_b200.fp8 import fp8_matmul, gated_ffn_fp8

    w = packed(256, 256, cuda_device)
    store = torch.empty((m + 1) * 256, dtype=torch.bfloat16, device=cuda_device)
    x = store[:m * 256].view(m, 256)
    x.copy_(activations(m, 256, cuda_device))
    for out in (x, store[256:].view(m, 256), store[8:8 + m * 256].view(m, 256)):
        if m > 1 or out.data_ptr() < x.data_ptr() + 512:
            with pytest.raises(ValueError):
                fp8_matmul(x, w, out=out)
    want = gated_ffn_fp8(x, w, w, w)
    assert gated_ffn_fp8(x, w, w, w, out=x) is x and torch.equal(x, want)


def test_layouts_of_operands(cuda_device):
    """Views, odd pitches, misaligned beginnings, scales of another type: the values decide."""
    import torch

    from qk_b200.fp8 import Fp8Rows, Fp8Weights, fp8_matmul, fp8_weights, gated_ffn_fp8, quantize_fp8, rms_norm_fp8

    x, w = activations(9, 384, cuda_device), packed(200, 384, cuda_device)
    want = fp8_matmul(x, w)
    wide = torch.zeros((9, 1000), dtype=torch.bfloat16, device=cuda_device)
    for at in (0, 8, 5):
        wide[:, at:at + 384] = x
        assert torch.equal(fp8_matmul(wide[:, at:at + 384], w), want)
    assert torch.equal(fp8_matmul(x.t().contiguous().t(), w), want)
    store = torch.zeros(200 * 401 + 7, dtype=torch.uint8, device=cuda_device)
    odd = store[7:].view(200, 401)[:, :384]
    odd.copy_(w.codes.view(torch.uint8))
    assert torch.equal(fp8_matmul(x, Fp8Weights(odd.view(torch.float8_e4m3fn), w.scales.double().t().contiguous().t())), want)
    laid = fp8_weights(odd.cpu(), w.scales.cpu(), cuda_device)
    assert torch.equal(fp8_matmul(x, laid), want) and laid.codes.stride(0) % 16 == 0
    rows = quantize_fp8(x)
    assert torch.equal(fp8_matmul(Fp8Rows(rows.codes[::2], rows.scales[:, ::2]), w), want[::2])
    out = torch.empty((9, 200), device=cuda_device)
    assert fp8_matmul(x.float(), w, out=out) is out and torch.equal(out.to(torch.bfloat16), want)
    assert fp8_matmul(x[:0], w).shape == (0, 200) and gated_ffn_fp8(x[:0], w, w, packed(8, 200, cuda_device)).shape == (0, 8)
    gamma = torch.ones(385, dtype=torch.bfloat16, device=cuda_device)[1:]
    got, _ = rms_norm_fp8(wide[:, 5:389], gamma)
    same, _ = rms_norm_fp8(x, gamma.clone())
    assert torch.equal(got.codes.float(), same.codes.float()) and torch.equal(got.scales, same.scales)
    assert rms_norm_fp8(x[:0], gamma)[0].codes.shape == (0, 384)


def test_non_finite_values_stay_in_their_rows(cuda_device):
    import torch

    from qk_b200.fp8 import fp8_matmul, gated_ffn_fp8

    for m in (4, 70, 600, 2000):  # the last in the wide form
        x, w = activations(m, 512, cuda_device), packed(700, 512, cuda_device)
        down = packed(64, 700, cuda_device)
        want, ffn = fp8_matmul(x, w), gated_ffn_fp8(x, w, w, down)
        x[1, 200] = float("nan")
        x[m - 1, 3] = float("inf")
        for got, good in ((fp8_matmul(x, w), want), (gated_ffn_fp8(x, w, w, down), ffn)):
            assert torch.isnan(got[1]).all() and torch.isnan(got[m - 1]).all()
            keep = [i for i in range(m) if i not in (1, m - 1)]
            assert torch.equal(got[keep], good[keep])


def test_rows_do_not_depend_on_their_neighbours(cuda_device):
    """Padding rows, whatever they hold, and the number of rows within a form change no bit of the others."""
    import torch

    from qk_b200.fp8 import fp8_matmul

    x, w = activations(64, 640, cuda_device), packed(1000, 640, cuda_device)
    want = fp8_matmul(x, w)
    y = x.clone()
    y[40:] = float("nan")
    assert torch.equal(fp8_matmul(y, w)[:40], want[:40])
    assert torch.equal(fp8_matmul(x[:50], w), want[:50])


def test_other_streams_threads_and_graphs(cuda_device):
    """Calls on several streams and from several threads at once, and two graphs replayed beside one another."""
    import threading

    import torch

    from qk_b200.fp8 import check_status, fp8_matmul, gated_ffn_fp8

    w, gate, down = packed(2048, 512, cuda_device), packed(640, 512, cuda_device, 2), packed(512, 640, cuda_device, 3)
    sizes = (1, 3, 20, 64, 100, 300)
    xs = [activations(m, 512, cuda_device, m) for m in sizes]

    def both(x):
        return fp8_matmul(x, w), gated_ffn_fp8(x, gate, gate, down)

    want = [both(x) for x in xs]
    torch.cuda.synchronize(cuda_device)
    bad = []

    def work(i):
        stream = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(stream):
            for _ in range(40):
                got = both(xs[i])
                if not all(torch.equal(g, e) for g, e in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    graphs, outs = [], []
    for x in xs[2:4]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([both(x) for _ in range(10)])
        graphs.append(graph)
    streams = [torch.cuda.Stream(cuda_device) for _ in graphs]
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize(cuda_device)
    for got, expected in zip(outs, want[2:4]):
        for pair in got:
            assert all(torch.equal(g, e) for g, e in zip(pair, expected))
    check_status(cuda_device)


def test_products_are_repeatable(cuda_device):
    """Sums are joined in a fixed order: equal calls give equal bits, wide and narrow."""
    import torch

    from qk_b200.fp8 import fp8_matmul, gated_fp8, quantize_fp8

    for m, k, n in ((1, 4096, 2048), (64, 2048, 9216), (2000, 2048, 2304)):
        x, w = quantize_fp8(activations(m, k, cuda_device)), packed(n, k, cuda_device)
        want, h = fp8_matmul(x, w, output_dtype=torch.float32), gated_fp8(x, w, w)
        for _ in range(30):
            assert torch.equal(fp8_matmul(x, w, output_dtype=torch.float32), want)
            again = gated_fp8(x, w, w)
            assert torch.equal(again.codes.view(torch.uint8), h.codes.view(torch.uint8)) and torch.equal(again.scales, h.scales)


def test_offsets_past_31_bits(cuda_device):
    """Rows whose values, codes and outputs lie more than 2^31 elements from the first."""
    import torch

    from qk_b200.fp8 import fp8_matmul, quantize_fp8, rms_norm_fp8

    rows, width = 600_000, 4096  # 2.5e9 values
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device=cuda_device)
    tail = activations(300, width, cuda_device)
    x[-300:] = tail
    got, want = quantize_fp8(x), quantize_fp8(tail)
    assert torch.equal(got.codes[-300:].float(), want.codes.float()) and torch.equal(got.scales[:, -300:], want.scales)
    w = packed(130, width, cuda_device)
    out = fp8_matmul(got, w)
    assert torch.equal(out[-300:], fp8_matmul(quantize_fp8(tail), w)) or np.abs(
        to_f32(out[-300:]) - to_f32(fp8_matmul(want, w))).max() <= 2.0 ** -7 * np.abs(to_f32(out[-300:])).max()
    assert not out[:1000].any()
    gamma = torch.ones(width, dtype=torch.bfloat16, device=cuda_device)
    normed, total = rms_norm_fp8(x, gamma, residual=x)
    small, _ = rms_norm_fp8(tail, gamma, residual=tail)
    assert torch.equal(normed.codes[-300:].float(), small.codes.float())
    assert torch.equal(total[-300:], (tail.float() * 2).to(torch.bfloat16))


def test_nothing_is_written_past_the_rows(cuda_device):
    """Codes, scales and outputs in buffers of other bytes: those between and behind the rows stay."""
    import torch

    from qk_b200 import _lib
    from qk_b200.fp8 import quantize_fp8

    def guarded(rows, ld, kind):
        store = torch.full(((rows + 1) * ld,), 0xAA, dtype=torch.uint8, device=cuda_device)
        return store, store.view(rows + 1, ld), kind

    P, st = _lib.ptr, _lib.stream_handle(cuda_device)
    for m, k, n in ((3, 133, 77), (40, 264, 130), (300, 1111, 1001), (2000, 300, 1290)):
        x, w = activations(m, k, cuda_device), packed(n, k, cuda_device)
        rows, ld = quantize_fp8(x), (max(k, n) + 47) // 16 * 16
        for name in ("qk_fp8_quantize", "qk_fp8_quantize_blocks"):
            store, codes, _ = guarded(m, ld, name)
            scales = torch.full((((k + 127) // 128) * m + 8,), 7.0, device=cuda_device)
            _lib.call(name, P(x), 1, k, m, k, P(store), ld, P(scales), st)
            assert (codes[:m, k:] == 0xAA).all() and (codes[m] == 0xAA).all() and (scales[-8:] == 7).all(), name
        store, codes, _ = guarded(m, ld, "gated")
        scales = torch.full((((n + 127) // 128) * m + 8,), 7.0, device=cuda_device)
        args = [P(rows.codes), rows.codes.stride(0), P(rows.scales), m, k] + [P(w.codes), w.codes.stride(0), P(w.scales)] * 2
        _lib.call("qk_fp8_gated", *args, n, P(store), ld, P(scales), st)
        assert (codes[:m, n:] == 0xAA).all() and (codes[m] == 0xAA).all() and (scales[-8:] == 7).all()
        for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
            out = torch.full((m * n + 64,), 7.0, dtype=dtype, device=cuda_device)
            _lib.call("qk_fp8_matmul", *args[:8], n, code, P(out), st)
            assert (out[m * n:] == 7).all()
