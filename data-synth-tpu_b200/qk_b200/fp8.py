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
_E4M3, _F32 = torch.float8_e4m3fn, torch.float32
_TYPES = {torch.bfloat16: _lib.QK_OUT_BF16, torch.float32: _lib.QK_OUT_F32}


class Fp8Rows(NamedTuple):
    """Quantised activations: value ``[m, k]`` is ``codes[m, k] * scales[k // 128, m]``."""

    codes: torch.Tensor   # float8_e4m3fn [M, K]
    scales: torch.Tensor  # FP32 [ceil(K / 128), M]


class Fp8Weights(NamedTuple):
    """Quantised weights: value ``[n, k]`` is ``codes[n, k] * scales[n // 128, k // 128]``."""

    codes: torch.Tensor   # float8_e4m3fn [N, K]
    scales: torch.Tensor  # FP32 [ceil(N / 128), ceil(K / 128)]


# The allocation that compiled graphs make, at half the cost of torch.empty_strided: on the current device only. A private
# function of torch, taken where it is there; dispatch modes do not see what it allocates.
_lean_empty = getattr(getattr(torch._C._dynamo, "guards", None), "_empty_strided_cuda", None)
_current = getattr(torch._C, "_cuda_getDevice", None)


def _empty(size, stride, dtype, index):
    if _lean_empty is not None and _current() == index:
        return _lean_empty(size, stride, dtype)
    return torch.empty_strided(size, stride, dtype=dtype, device=torch.device("cuda", index))


def _blocks(n):
    return (n + 127) // 128


def _empty_rows(rows, width, index):
    """:class:`Fp8Rows` to be written; rows of codes begin on 16 bytes."""
    pitch = (width + 15) // 16 * 16
    return Fp8Rows(_empty((rows, width), (pitch, 1), _E4M3, index), _empty((_blocks(width), rows), (rows, 1), _F32, index)), pitch


def _quantised(codes, scales, by_rows, name):
    """What a product reads of Fp8Rows (``by_rows``) or Fp8Weights: ``(codes, bytes from row to row, scales)``.
    Copied only where it is not laid out as the kernels read it: rows of codes that begin on 16 bytes,
    scales contiguous."""
    if not isinstance(codes, torch.Tensor) or codes.dtype != _E4M3 or codes.dim() != 2:
        raise TypeError(f"{name} must hold float8_e4m3fn codes, a matrix")
    index = codes.get_device()
    if index < 0:
        raise ValueError("expected CUDA tensors")
    rows, width = codes.shape
    if scales.shape != ((_blocks(width), rows) if by_rows else (_blocks(rows), _blocks(width))):
        raise ValueError(f"the scales of {name} do not match its codes, one for each block of 128")
    pitch, step = codes.stride()
    if pitch % 16 or pitch < width or step != 1 or codes.data_ptr() % 16:
        pitch = (width + 15) // 16 * 16
        codes = torch.empty_strided((rows, width), (pitch, 1), dtype=_E4M3, device=codes.device).copy_(codes)
    if scales.dtype != _F32 or scales.get_device() != index:
        scales = scales.to(device=codes.device, dtype=_F32)
    return codes, pitch, scales if scales.is_contiguous() else scales.contiguous()


def _weights(weights, k, index, name):
    """``weights`` of a product of ``k`` columns on device ``index``: ``(rows, address, bytes from row to row,
    address of the scales)``, and the tensors, which have to live until the call is made."""
    codes, scales = weights
    if codes.dtype is not _E4M3 or k % 16 or not (codes.is_contiguous() and scales.is_contiguous()) or scales.dtype is not _F32 \
            or codes.data_ptr() % 16 or scales.get_device() != index:
        codes, pitch, scales = _quantised(codes, scales, False, name)
    else:
        pitch = k
    n, width = codes.shape
    if width != k or n < 1 or codes.get_device() != index:
        raise ValueError(f"{name} must be [N, {k}] on the device of x")
    if scales.shape != ((n + 127) // 128, (k + 127) // 128):
        raise ValueError(f"the scales of {name} do not match its codes, one for each block of 128")
    return n, codes.data_ptr(), pitch, scales.data_ptr(), (codes, scales)


def _matrix(x, name):
    """``x`` BF16 or FP32 ``[rows, width]`` with dense rows: ``(x, rows, width, type code, stride, device
    number)``."""
    shape = x.shape if isinstance(x, torch.Tensor) else ()
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{name} must be a BF16 or FP32 matrix")
    rows, width = shape
    code = _TYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{name} must be BF16 or FP32")
    index = x.get_device()
    if index < 0:
        raise ValueError("expected CUDA tensors")
    if x.is_contiguous():
        return x, rows, width, code, width, index
    if width > 1 and x.stride(1) != 1 or rows > 1 and x.stride(0) < width:
        return x.contiguous(), rows, width, code, width, index
    return x, rows, width, code, max(x.stride(0), width), index


_needs = {}


def _room(name, index, code, m, k, n, x, stride):
    """``(x, stride, workspace, its bytes)`` of a product from rows of BF16 or FP32: where the product
    quantises them itself, they begin on 16 bytes."""
    key = (name, index, code, m, k, n)
    need = _needs.get(key)
    if need is None:
        if len(_needs) > 4096:
            _needs.clear()
        with torch.cuda.device(index):
            need = _needs[key] = int(getattr(_lib.load(), name)(code, m, k, n))
    if k % 8 == 0 and (x.data_ptr() % 16 or stride * x.element_size() % 16):
        x, stride = x.clone(memory_format=torch.contiguous_format), k
    return x, stride, _empty((need,), (1,), torch.uint8, index) if need else None, need


def quantize_fp8(x):
    """``x`` BF16 or FP32 ``[M, K]`` (rows may be strided) -> :class:`Fp8Rows`. A block of a row with
    the largest magnitude ``m`` (at least 2^-100) has the scale ``m / 448`` and the codes
    ``e4m3(448 x / m)``. A block that holds an infinity or a NaN has no finite values."""
    x, rows, width, code, stride, index = _matrix(x, "x")
    out, pitch = _empty_rows(rows, width, index)
    _lib.call_at(index, "qk_fp8_quantize", x.data_ptr(), code, stride, rows, width, out.codes.data_ptr(), pitch,
                 out.scales.data_ptr())
    return out


def pack_fp8(weight):
    """``weight`` BF16 or FP32 ``[N, K]`` -> :class:`Fp8Weights`, by the rule of :func:`quantize_fp8`
    for blocks of 128 x 128."""
    weight, rows, width, code, stride, index = _matrix(weight, "weight")
    pitch = (width + 15) // 16 * 16
    codes = torch.empty_strided((rows, width), (pitch, 1), dtype=_E4M3, device=weight.device)
    scales = torch.empty((_blocks(rows), _blocks(width)), dtype=_F32, device=weight.device)
    _lib.call_at(index, "qk_fp8_quantize_blocks", weight.data_ptr(), code, stride, rows, width, codes.data_ptr(), pitch,
                 scales.data_ptr())
    return Fp8Weights(codes, scales)


def fp8_weights(codes, scales, device=None):
    """A checkpoint's codes ``[N, K]`` (float8_e4m3fn, or uint8 of the same bits) and scales
    ``[ceil(N / 128), ceil(K / 128)]`` (what the codes are multiplied by) on ``device``, laid out once
    so that calls need not copy them."""
    device = torch.device(device if device is not None else codes.device if codes.is_cuda else "cuda")
    if codes.dtype == torch.uint8:
        codes = codes.view(_E4M3)
    codes, _, scales = _quantised(codes.to(device), scales, False, "the weights")
    return Fp8Weights(codes, scales)


def _output(out, m, n, dtype, index, *inputs):
    """``out``, or a new output; it must not share memory with ``inputs``, matrices of dense rows."""
    if out is None:
        return _empty((m, n), (n, 1), dtype, index)
    if out.dtype != dtype or out.shape != (m, n) or out.get_device() != index or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {[m, n]} on the device of x")
    for x in inputs if m else ():
        first, size = x.data_ptr(), ((x.shape[0] - 1) * x.stride(0) + x.shape[1]) * x.element_size()
        if first < out.data_ptr() + out.nbytes and out.data_ptr() < first + size:
            raise ValueError("out must not share memory with x, which is read while out is written")
    return out


def fp8_matmul(x, weights, *, output_dtype=None, out=None):
    """``x @ weights.T`` as ``[M, N]`` BF16 (default) or FP32 (``output_dtype``). ``x`` is BF16 or FP32
    ``[M, K]``, quantised in the call, or :class:`Fp8Rows`. Products of codes are exact, sums FP32. ``out``
    must not share memory with ``x`` (codes or scales)."""
    dtype = output_dtype or (torch.bfloat16 if out is None else out.dtype)
    out_code = _TYPES.get(dtype)
    if out_code is None:
        raise ValueError("output_dtype must be BF16 or FP32")
    if isinstance(x, Fp8Rows):
        codes, pitch, scales = _quantised(x.codes, x.scales, True, "x")
        m, k = codes.shape
        index = codes.get_device()
        n, w, w_pitch, w_scales, _keep = _weights(weights, k, index, "weights")
        out = _output(out, m, n, dtype, index, codes, scales)
        _lib.call_at(index, "qk_fp8_matmul", codes.data_ptr(), pitch, scales.data_ptr(), m, k, w, w_pitch, w_scales, n,
                     out_code, out.data_ptr())
        return out
    x, m, k, code, stride, index = _matrix(x, "x")
    n, w, w_pitch, w_scales, _keep = _weights(weights, k, index, "weights")
    out = _output(out, m, n, dtype, index, x)
    x, stride, room, need = _room("qk_fp8_linear_workspace_bytes", index, code, m, k, n, x, stride)
    _lib.call_at(index, "qk_fp8_linear", x.data_ptr(), code, stride, m, k, w, w_pitch, w_scales, n,
                 out_code, out.data_ptr(), room.data_ptr() if need else None, need)
    return out


def gated_fp8(x, gate, up):
    """``silu(x gate^T) * (x up^T)`` as :class:`Fp8Rows` ``[M, I]``, quantised from FP32 by the rule of
    :func:`quantize_fp8`: ``x`` as for :func:`fp8_matmul`, ``gate`` and ``up`` ``[I, K]``."""
    x = x if isinstance(x, Fp8Rows) else quantize_fp8(x)
    codes, pitch, scales = _quantised(x.codes, x.scales, True, "x")
    m, k = codes.shape
    index = codes.get_device()
    inner, g, g_pitch, g_scales, _keep_g = _weights(gate, k, index, "gate")
    n, u, u_pitch, u_scales, _keep_u = _weights(up, k, index, "up")
    if n != inner:
        raise ValueError("gate and up must be [I, K]")
    h, h_pitch = _empty_rows(m, inner, index)
    _lib.call_at(index, "qk_fp8_gated", codes.data_ptr(), pitch, scales.data_ptr(), m, k, g, g_pitch, g_scales,
                 u, u_pitch, u_scales, inner, h.codes.data_ptr(), h_pitch,
                 h.scales.data_ptr())
    return h


def gated_ffn_fp8(x, gate, up, down, *, out=None):
    """A gated feed-forward block, ``(silu(x gate^T) * (x up^T)) down^T`` as BF16 ``[M, H]``: the product
    of :func:`gated_fp8` with ``down`` ``[H, I]``. ``out`` may be ``x``."""
    if isinstance(x, Fp8Rows):
        return fp8_matmul(gated_fp8(x, gate, up), down, out=out, output_dtype=torch.bfloat16)
    x, m, k, code, stride, index = _matrix(x, "x")
    inner, g, g_pitch, g_scales, _keep_g = _weights(gate, k, index, "gate")
    n, u, u_pitch, u_scales, _keep_u = _weights(up, k, index, "up")
    if n != inner:
        raise ValueError("gate and up must be [I, K]")
    n, d, d_pitch, d_scales, _keep_d = _weights(down, inner, index, "down")
    out = _output(out, m, n, torch.bfloat16, index)
    x, stride, room, need = _room("qk_fp8_ffn_workspace_bytes", index, code, m, k, inner, x, stride)
    _lib.call_at(index, "qk_fp8_ffn", x.data_ptr(), code, stride, m, k, g, g_pitch, g_scales, u, u_pitch, u_scales, inner, d,
                 d_pitch, d_scales, n, out.data_ptr(), room.data_ptr() if need else None, need)
    return out


def _dense(t):
    """``t`` contiguous and 16-byte aligned."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def rms_norm_fp8(x, gamma, eps=1e-6, *, residual=None):
    """The residual add and RMSNorm of BF16 ``x`` ``[M, H]`` (``qwen38_tpu/math.py:27-31``), quantised:
    ``(Fp8Rows of rms(s) * gamma, s)`` with ``s = bf16(x + residual)``, or ``(Fp8Rows of rms(x) * gamma,
    None)`` without a residual. The norm is not rounded before its codes. ``H``: a multiple of 8, 8192 at
    most."""
    shape = x.shape
    if x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16 or len(shape) != 2 or gamma.shape != shape[1:]:
        raise TypeError("x and gamma must be BF16, [M, H] and [H]")
    rows, width = shape
    index = x.get_device()
    if index < 0:
        raise ValueError("expected CUDA tensors")
    if gamma.get_device() != index:
        raise ValueError("gamma must be on the device of x")
    x, gamma = _dense(x), _dense(gamma)
    total = y = kept = None
    if residual is not None:
        if residual.dtype != torch.bfloat16 or residual.shape != shape or residual.get_device() != index:
            raise ValueError("residual must be BF16 of x's shape on its device")
        residual = _dense(residual)
        total = _empty((rows, width), (width, 1), torch.bfloat16, index)
        y, kept = residual.data_ptr(), total.data_ptr()
    out, pitch = _empty_rows(rows, width, index)
    _lib.call_at(index, "qk_fp8_rms_norm", x.data_ptr(), y, gamma.data_ptr(), rows, width, eps, kept, out.codes.data_ptr(),
                 pitch, out.scales.data_ptr())
    return out, total


def check_status(device=None):
    """Raise what products on the device reported (a bounded wait that gave up), in graphs and on other
    streams too as far as they have run; synchronises the current stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    _lib.call_on(device, "qk_fp8_check")


__all__ = ["BLOCK", "Fp8Rows", "Fp8Weights", "check_status", "fp8_matmul", "fp8_weights", "gated_ffn_fp8", "gated_fp8",
           "pack_fp8", "quantize_fp8", "rms_norm_fp8"]
