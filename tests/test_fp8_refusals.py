"""FP8 dense path: what its entry points refuse, before any launch (no GPU)."""

import ctypes

import pytest
import torch

E4M3 = torch.float8_e4m3fn


def p(address):
    return ctypes.c_void_p(address)


GOOD = dict(
    qk_fp8_quantize=[p(64), 1, 256, 2, 256, p(256), 256, p(16), None],
    qk_fp8_quantize_blocks=[p(64), 0, 256, 2, 256, p(256), 256, p(16), None],
    qk_fp8_rms_norm=[p(64), p(128), p(64), 2, 256, 1e-6, p(64), p(256), 256, p(16), None],
    qk_fp8_matmul=[p(64), 256, p(16), 2, 256, p(64), 256, p(16), 128, 1, p(64), None],
    qk_fp8_gated=[p(64), 256, p(16), 2, 256, p(64), 256, p(16), p(64), 256, p(16), 128, p(64), 128, p(16), None],
    qk_fp8_linear=[p(64), 1, 256, 300, 256, p(64), 256, p(16), 128, 1, p(64), p(256), 1 << 30, None],
    qk_fp8_ffn=[p(64), 1, 256, 2, 256, p(64), 256, p(16), p(64), 256, p(16), 128, p(64), 128, p(16), 256, p(64), p(256), 1 << 30,
                None],
)

# entry point, argument, a value that it refuses
BAD = [
    ("qk_fp8_quantize", 1, 2), ("qk_fp8_quantize", 2, 255), ("qk_fp8_quantize", 3, -1), ("qk_fp8_quantize", 4, 0),
    ("qk_fp8_quantize", 6, 255), ("qk_fp8_quantize", 6, 240), ("qk_fp8_quantize", 0, p(0)), ("qk_fp8_quantize", 0, p(65)),
    ("qk_fp8_quantize", 5, p(8)), ("qk_fp8_quantize", 7, p(18)), ("qk_fp8_quantize", 3, 1 << 40),
    ("qk_fp8_quantize_blocks", 1, 30), ("qk_fp8_quantize_blocks", 2, 128), ("qk_fp8_quantize_blocks", 3, 65536 * 128),
    ("qk_fp8_quantize_blocks", 7, p(0)),
    ("qk_fp8_rms_norm", 4, 250), ("qk_fp8_rms_norm", 4, 8200), ("qk_fp8_rms_norm", 4, 0), ("qk_fp8_rms_norm", 0, p(68)),
    ("qk_fp8_rms_norm", 6, p(0)), ("qk_fp8_rms_norm", 8, 248), ("qk_fp8_rms_norm", 3, -1),
    ("qk_fp8_matmul", 1, 248), ("qk_fp8_matmul", 1, 128), ("qk_fp8_matmul", 3, -1), ("qk_fp8_matmul", 4, 0), ("qk_fp8_matmul", 6, 264),
    ("qk_fp8_matmul", 8, 0), ("qk_fp8_matmul", 9, 30), ("qk_fp8_matmul", 0, p(72)), ("qk_fp8_matmul", 5, p(0)),
    ("qk_fp8_matmul", 10, p(65)), ("qk_fp8_matmul", 7, p(17)), ("qk_fp8_matmul", 3, 1 << 31),
    ("qk_fp8_gated", 13, 120), ("qk_fp8_gated", 12, p(72)), ("qk_fp8_gated", 14, p(0)), ("qk_fp8_gated", 8, p(0)),
    ("qk_fp8_gated", 9, 248), ("qk_fp8_gated", 11, 0),
    ("qk_fp8_linear", 1, 7), ("qk_fp8_linear", 2, 100), ("qk_fp8_linear", 0, p(65)), ("qk_fp8_linear", 9, 5),
    ("qk_fp8_linear", 11, p(8)),
    ("qk_fp8_ffn", 13, 136), ("qk_fp8_ffn", 15, 0), ("qk_fp8_ffn", 16, p(65)), ("qk_fp8_ffn", 12, p(0)), ("qk_fp8_ffn", 0, p(72)),
]


@pytest.mark.parametrize("name,at,value", BAD)
def test_entry_points_refuse(name, at, value):
    from qk_b200 import _lib

    args = list(GOOD[name])
    args[at] = value
    assert getattr(_lib.load(), name)(*args) == _lib.QK_ERR_INVALID_ARGUMENT, _lib.last_error()


def test_workspaces_are_checked():
    from qk_b200 import _lib

    lib = _lib.load()
    need = lib.qk_fp8_linear_workspace_bytes(1, 300, 256, 128)
    assert need >= 300 * 256 + 2 * 300 * 4
    args = list(GOOD["qk_fp8_linear"])
    args[12] = need - 1
    assert lib.qk_fp8_linear(*args) == _lib.QK_ERR_WORKSPACE
    args[11:13] = [None, 0]
    assert lib.qk_fp8_linear(*args) == _lib.QK_ERR_WORKSPACE
    # few rows of BF16 need none, FP32 and odd widths do
    assert lib.qk_fp8_linear_workspace_bytes(1, 2, 2048, 9216) == 0
    assert lib.qk_fp8_linear_workspace_bytes(0, 2, 2048, 9216) > 0
    assert lib.qk_fp8_linear_workspace_bytes(1, 2, 2047, 9216) > 0
    args = list(GOOD["qk_fp8_ffn"])
    args[18] = lib.qk_fp8_ffn_workspace_bytes(1, 2, 256, 128) - 1
    assert lib.qk_fp8_ffn(*args) == _lib.QK_ERR_WORKSPACE


def test_nothing_to_do_is_no_error():
    from qk_b200 import _lib

    for name, at in (("qk_fp8_quantize", 3), ("qk_fp8_quantize_blocks", 3), ("qk_fp8_rms_norm", 3), ("qk_fp8_matmul", 3),
                     ("qk_fp8_gated", 3), ("qk_fp8_linear", 3), ("qk_fp8_ffn", 3)):
        args = [None if isinstance(a, ctypes.c_void_p) else a for a in GOOD[name]]
        args[at] = 0
        assert getattr(_lib.load(), name)(*args) == _lib.QK_OK, (name, _lib.last_error())


def test_python_calls_refuse():
    from qk_b200.decoder import StackConfig, SyntheticDecoder
    from qk_b200.fp8 import (Fp8Rows, Fp8Weights, fp8_matmul, fp8_weights, gated_ffn_fp8, gated_fp8, pack_fp8, quantize_fp8,
                             rms_norm_fp8)

    x, codes = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros((128, 256), dtype=torch.uint8).view(E4M3)
    w = Fp8Weights(codes, torch.ones((1, 2)))
    rows = Fp8Rows(codes[:4], torch.ones((2, 4)))
    for call in (lambda: quantize_fp8(x), lambda: pack_fp8(x), lambda: fp8_matmul(x, w), lambda: fp8_matmul(rows, w),
                 lambda: gated_fp8(x, w, w), lambda: gated_ffn_fp8(x, w, w, w), lambda: rms_norm_fp8(x, x[0])):
        with pytest.raises(ValueError):
            call()  # not on a GPU
    for call in (lambda: quantize_fp8(x[0]), lambda: quantize_fp8(x[:, :0]), lambda: fp8_matmul([1.0], w),
                 lambda: fp8_matmul(x, w, output_dtype=torch.float16)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: quantize_fp8(x.to(torch.float16)), lambda: fp8_matmul(Fp8Rows(x, rows.scales), w),
                 lambda: rms_norm_fp8(x, x[0, :8]), lambda: rms_norm_fp8(x.float(), x[0]),
                 lambda: fp8_weights(x, w.scales, device="cpu")):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        SyntheticDecoder(StackConfig(layers=0, dense="fp4"), "cpu")


@pytest.mark.parametrize("m,k,n", [(0, 128, 128), (-5, 128, 128), (4, 0, 128), (4, 128, -1), (1 << 62, 1 << 62, 4), (1 << 62, 128, 1 << 62),
                                   ((1 << 63) - 1, 128, (1 << 63) - 1), (4, (1 << 63) - 1, 4)])
def test_sizes_that_no_call_takes_need_no_workspace(m, k, n):
    from qk_b200 import _lib

    lib = _lib.load()
    for dtype in (0, 1):
        assert lib.qk_fp8_linear_workspace_bytes(dtype, m, k, n) == 0
        assert lib.qk_fp8_ffn_workspace_bytes(dtype, m, k, n) == 0


@pytest.mark.parametrize("name,at", [("qk_fp8_quantize", 3), ("qk_fp8_quantize_blocks", 3), ("qk_fp8_rms_norm", 3), ("qk_fp8_matmul", 3),
                                     ("qk_fp8_matmul", 4), ("qk_fp8_matmul", 8), ("qk_fp8_linear", 3), ("qk_fp8_gated", 11),
                                     ("qk_fp8_ffn", 15)])
def test_the_largest_sizes_are_refused(name, at):
    from qk_b200 import _lib

    args = list(GOOD[name])
    args[at] = (1 << 63) - 1
    assert getattr(_lib.load(), name)(*args) == _lib.QK_ERR_INVALID_ARGUMENT, _lib.last_error()
