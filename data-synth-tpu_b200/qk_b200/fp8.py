"""FP8 dense path: projections whose weights and activations are e4m3 codes with an FP32 scale for
each block of 128 (activations: per row and 128 columns; weights: per 128 x 128, the layout of block
FP8 checkpoints).

::

    w = pack_fp8(weight)                           # or fp8_weights(codes, scales) of a checkpoint
    y = fp8_matmul(x, w)                           # x BF16 [M, K], quantised in the call
    rows, x = rms_norm_fp8(x, gamma, residual=y)   # the residual add, the norm and the quantisation
    q = fp8_matmul(rows, w)
    y = gated_ffn_fp8(x, gate, up, down)

The reference's dense projections are BF16 (``qwen38_tpu/math.py:10-16``); these stand beside
:func:`~qk_b200.packed.linear_bf16` and the packed products.
"""

from typing import NamedTuple

import torch

from . import _lib

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_TYPES = {torch.bfloat16: _lib.QK_OUT_BF16, torch.float32: _lib.QK_OUT_F32}


class Fp8Rows(NamedTuple):
    """Quantised activations: value ``[m, k]`` is ``codes[m, k] * scales[k // 128, m]``."""

    codes: torch.Tensor   # float8_e4m3fn [M, K]
    scales: torch.Tensor  # FP32 [ceil(K / 128), M]


class Fp8Weights(NamedTuple):
    """Quantised weights: value ``[n, k]`` is ``codes[n, k] * scales[n // 128, k // 128]``."""

    codes: torch.Tensor   # float8_e4m3fn [N, K]
    scales: torch.Tensor  # FP32 [ceil(N / 128), ceil(K / 128)]


def _blocks(n):
    return -(-n // BLOCK)


def _empty_rows(like, rows, width):
    """:class:`Fp8Rows` to be written, on the device of ``like``; rows of codes begin on 16 bytes."""
    pitch = (width + 15) // 16 * 16
    codes = like.new_empty((rows, pitch), dtype=_E4M3)
    return (Fp8Rows(codes if pitch == width else codes[:, :width], like.new_empty((_blocks(width), rows), dtype=torch.float32)),
            pitch)


def _codes(codes, name):
    """Codes as the products read them, and the bytes from row to row; copied only where their rows
    are not evenly spaced on 16-byte boundaries."""
    if codes.dtype != _E4M3 or codes.dim() != 2:
        raise TypeError(f"{name} must hold float8_e4m3fn codes, a matrix")
    if not codes.is_cuda:
        raise ValueError("expected CUDA tensors")
    rows, width = codes.shape
    pitch = codes.stride(0)
    if rows == 1 and pitch < width:
        pitch = (width + 15) // 16 * 16
    if pitch % 16 or pitch < width or codes.data_ptr() % 16 or (width > 1 and codes.stride(1) != 1):
        pitch = (width + 15) // 16 * 16
        fresh = codes.new_empty((rows, pitch))[:, :width]
        fresh.copy_(codes)
        return fresh, pitch
    return codes, pitch


def _scales(scales, shape, device, name):
    if scales.shape != shape:
        raise ValueError(f"{name} must have scales {list(shape)}, got {list(scales.shape)}")
    if scales.dtype != torch.float32 or scales.device != device:
        scales = scales.to(device=device, dtype=torch.float32)
    return scales if scales.is_contiguous() else scales.contiguous()


def _matrix(x, name):
    """``x`` BF16 or FP32 ``[rows, width]`` with dense rows: ``(x, type code, stride)``."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{name} must be a BF16 or FP32 matrix")
    code = _TYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{name} must be BF16 or FP32")
    if not x.is_cuda:
        raise ValueError("expected CUDA tensors")
    if x.is_contiguous():
        return x, code, x.shape[1]
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        return x.contiguous(), code, x.shape[1]
    return x, code, max(x.stride(0), x.shape[1])


def _aligned(x, name):
    """The same with rows that begin on 16 bytes if those of a fresh tensor do."""
    x, code, stride = _matrix(x, name)
    if x.data_ptr() % 16 or stride * x.element_size() % 16:
        return x.clone(memory_format=torch.contiguous_format), code, x.shape[1]
    return x, code, stride


_needs = {}


def _workspace(name, key, device):
    """``(workspace, bytes)`` of a call on ``device``, from the current stream's memory."""
    need = _needs.get((name, key))
    if need is None:
        with torch.cuda.device(device):
            need = _needs[name, key] = int(getattr(_lib.load(), name)(*key))
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


def quantize_fp8(x):
    """``x`` BF16 or FP32 ``[M, K]`` (rows may be strided) -> :class:`Fp8Rows`. A block of a row with
    the largest magnitude ``m`` (at least 2^-100) has the scale ``m / 448`` and the codes
    ``e4m3(448 x / m)``. A block that holds an infinity or a NaN has no finite values."""
    x, code, stride = _matrix(x, "x")
    rows, width = x.shape
    out, pitch = _empty_rows(x, rows, width)
    _lib.call_on(x.device, "qk_fp8_quantize", x.data_ptr(), code, stride, rows, width, out.codes.data_ptr(), pitch,
                 out.scales.data_ptr())
    return out


def pack_fp8(weight):
    """``weight`` BF16 or FP32 ``[N, K]`` -> :class:`Fp8Weights`, by the rule of :func:`quantize_fp8`
    for blocks of 128 x 128."""
    weight, code, stride = _matrix(weight, "weight")
    rows, width = weight.shape
    pitch = (width + 15) // 16 * 16
    codes = weight.new_empty((rows, pitch), dtype=_E4M3)[:, :width]
    scales = weight.new_empty((_blocks(rows), _blocks(width)), dtype=torch.float32)
    _lib.call_on(weight.device, "qk_fp8_quantize_blocks", weight.data_ptr(), code, stride, rows, width, codes.data_ptr(),
                 pitch, scales.data_ptr())
    return Fp8Weights(codes, scales)


def fp8_weights(codes, scales, device=None):
    """A checkpoint's codes ``[N, K]`` (float8_e4m3fn, or uint8 of the same bits) and scales
    ``[ceil(N / 128), ceil(K / 128)]`` (what the codes are multiplied by) on ``device``, laid out once
    so that calls need not copy them."""
    device = torch.device(device or (codes.device if codes.is_cuda else "cuda"))
    if codes.dtype == torch.uint8:
        codes = codes.view(_E4M3)
    codes, _ = _codes(codes.to(device), "codes")
    shape = (_blocks(codes.shape[0]), _blocks(codes.shape[1]))
    return Fp8Weights(codes, _scales(scales, shape, codes.device, "the weights"))


def _operand(weights, k, device, name):
    """``weights`` as a product of ``k`` columns on ``device`` reads them: ``(rows, codes, pitch, scales)``."""
    codes, pitch = _codes(weights.codes, name)
    n, width = codes.shape
    if width != k or n < 1 or codes.device != device:
        raise ValueError(f"{name} must be [N, {k}] on the device of x")
    return n, codes, pitch, _scales(weights.scales, (_blocks(n), _blocks(k)), device, name)


def _rows(x):
    """Quantised activations as a product reads them: ``(codes, pitch, scales)``."""
    codes, pitch = _codes(x.codes, "x")
    return codes, pitch, _scales(x.scales, (_blocks(codes.shape[1]), codes.shape[0]), codes.device, "x")


def _output(out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.dtype != dtype or out.shape != shape or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {list(shape)} on the device of x")
    return out


def fp8_matmul(x, weights, *, output_dtype=None, out=None):
    """``x @ weights.T`` as ``[M, N]`` BF16 (default) or FP32 (``output_dtype``). ``x`` is BF16 or FP32
    ``[M, K]``, quantised in the call, or :class:`Fp8Rows`. Products of codes are exact, sums FP32."""
    dtype = output_dtype or (torch.bfloat16 if out is None else out.dtype)
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("output_dtype must be BF16 or FP32")
    out_code = _lib.QK_OUT_F32 if dtype == torch.float32 else _lib.QK_OUT_BF16
    if isinstance(x, Fp8Rows):
        codes, pitch, scales = _rows(x)
        (m, k), device = codes.shape, codes.device
        n, w, w_pitch, w_scales = _operand(weights, k, device, "weights")
        out = _output(out, (m, n), dtype, device)
        _lib.call_on(device, "qk_fp8_matmul", codes.data_ptr(), pitch, scales.data_ptr(), m, k, w.data_ptr(), w_pitch,
                     w_scales.data_ptr(), n, out_code, out.data_ptr())
        return out
    x, code, stride = _aligned(x, "x")
    (m, k), device = x.shape, x.device
    n, w, w_pitch, w_scales = _operand(weights, k, device, "weights")
    out = _output(out, (m, n), dtype, device)
    room, need = _workspace("qk_fp8_linear_workspace_bytes", (code, m, k, n), device)
    _lib.call_on(device, "qk_fp8_linear", x.data_ptr(), code, stride, m, k, w.data_ptr(), w_pitch, w_scales.data_ptr(), n,
                 out_code, out.data_ptr(), room.data_ptr() if need else None, need)
    return out


def gated_fp8(x, gate, up):
    """``silu(x gate^T) * (x up^T)`` as :class:`Fp8Rows` ``[M, I]``, quantised from FP32 by the rule of
    :func:`quantize_fp8`: ``x`` as for :func:`fp8_matmul`, ``gate`` and ``up`` ``[I, K]``."""
    codes, pitch, scales = _rows(x if isinstance(x, Fp8Rows) else quantize_fp8(x))
    (m, k), device = codes.shape, codes.device
    inner, g, g_pitch, g_scales = _operand(gate, k, device, "gate")
    n, u, u_pitch, u_scales = _operand(up, k, device, "up")
    if n != inner:
        raise ValueError("gate and up must be [I, K]")
    h, h_pitch = _empty_rows(codes, m, inner)
    _lib.call_on(device, "qk_fp8_gated", codes.data_ptr(), pitch, scales.data_ptr(), m, k, g.data_ptr(), g_pitch,
                 g_scales.data_ptr(), u.data_ptr(), u_pitch, u_scales.data_ptr(), inner, h.codes.data_ptr(), h_pitch,
                 h.scales.data_ptr())
    return h


def gated_ffn_fp8(x, gate, up, down, *, out=None):
    """A gated feed-forward block, ``(silu(x gate^T) * (x up^T)) down^T`` as BF16 ``[M, H]``: the product
    of :func:`gated_fp8` with ``down`` ``[H, I]``."""
    if isinstance(x, Fp8Rows):
        return fp8_matmul(gated_fp8(x, gate, up), down, out=out, output_dtype=torch.bfloat16)
    x, code, stride = _aligned(x, "x")
    (m, k), device = x.shape, x.device
    inner, g, g_pitch, g_scales = _operand(gate, k, device, "gate")
    n, u, u_pitch, u_scales = _operand(up, k, device, "up")
    if n != inner:
        raise ValueError("gate and up must be [I, K]")
    n, d, d_pitch, d_scales = _operand(down, inner, device, "down")
    out = _output(out, (m, n), torch.bfloat16, device)
    room, need = _workspace("qk_fp8_ffn_workspace_bytes", (code, m, k, inner), device)
    _lib.call_on(device, "qk_fp8_ffn", x.data_ptr(), code, stride, m, k, g.data_ptr(), g_pitch, g_scales.data_ptr(),
                 u.data_ptr(), u_pitch, u_scales.data_ptr(), inner, d.data_ptr(), d_pitch, d_scales.data_ptr(), n, out.data_ptr(),
                 room.data_ptr() if need else None, need)
    return out


def rms_norm_fp8(x, gamma, eps=1e-6, *, residual=None):
    """The residual add and RMSNorm of BF16 ``x`` ``[M, H]`` (``qwen38_tpu/math.py:27-31``), quantised:
    ``(Fp8Rows of rms(s) * gamma, s)`` with ``s = bf16(x + residual)``, or ``(Fp8Rows of rms(x) * gamma,
    None)`` without a residual. The norm is not rounded before its codes. ``H``: a multiple of 8, 8192 at
    most."""
    if x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16 or x.dim() != 2 or gamma.shape != x.shape[1:]:
        raise TypeError("x and gamma must be BF16, [M, H] and [H]")
    (rows, width), device = x.shape, x.device
    if gamma.device != device or residual is not None and residual.device != device:
        raise ValueError("gamma and residual must be on the device of x")
    if residual is not None and (residual.dtype != torch.bfloat16 or residual.shape != x.shape):
        raise ValueError("residual must be BF16 of x's shape")
    x, gamma = _dense(x), _dense(gamma)
    out, pitch = _empty_rows(x, rows, width)
    total = y = None
    if residual is not None:
        residual = _dense(residual)
        total = torch.empty_like(x)
        y, kept = residual.data_ptr(), total.data_ptr()
    _lib.call_on(device, "qk_fp8_rms_norm", x.data_ptr(), y, gamma.data_ptr(), rows, width, eps, kept if y else None,
                 out.codes.data_ptr(), pitch, out.scales.data_ptr())
    return out, total


def _dense(t):
    """``t`` contiguous and 16-byte aligned."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def check_status(device=None):
    """Raise what products on the device reported (a bounded wait that gave up), in graphs and on other
    streams too as far as they have run; synchronises the current stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    _lib.call_on(device, "qk_fp8_check")


__all__ = ["BLOCK", "Fp8Rows", "Fp8Weights", "check_status", "fp8_matmul", "fp8_weights", "gated_ffn_fp8", "gated_fp8",
           "pack_fp8", "quantize_fp8", "rms_norm_fp8"]
