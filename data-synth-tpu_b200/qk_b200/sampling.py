"""Logits before the choice: penalties for repeated tokens, biases, temperature, grammar masks.

The reference's decoding is greedy (``qwen38_tpu/run.py:46-55``); :func:`process_logits` makes
the logits that a request's sampling rules ask for, to be followed by
:func:`~qk_b200.decoder.checked_argmax` or a draw.
"""

import ctypes

import torch

from . import _lib
from .attention_cache import _dtype_code
from .paged import _array


def process_logits(logits, *, history=None, history_lengths=None, prompt_lengths=None, repetition=None,
                   frequency=None, presence=None, temperature=None, bias_ids=None, bias=None, mask=None, drafts=None,
                   ancestors=None, out=None):
    """``logits`` BF16 or FP32 ``[B, V]``, or ``[B, N, V]`` with a row for every node of a draft
    tree -> FP32 of the same shape (``out`` may be the FP32 input). For every token of a row, in
    this order: if the token is in the context, ``x / repetition`` where ``x > 0`` and ``x *
    repetition`` elsewhere; ``x - frequency * n - presence * [n > 0]``; ``x + bias``; ``x /
    temperature``; ``-inf`` where the mask's bit is 0.

    ``history`` int32 ``[B, L]`` with ``history_lengths`` ``[B]`` holds each request's tokens, of
    which the first ``prompt_lengths[b]`` (default 0) are its prompt; ``n`` counts the generated
    ones, and with ``drafts`` int32 ``[B, N]`` and ``ancestors`` int64 ``[B, N]``
    (:func:`~qk_b200.paged.plan_step`) the drafted ones on the row's path. ``repetition``,
    ``frequency``, ``presence``, ``temperature`` (above 0): FP32 ``[B]``. ``bias_ids`` int32 and
    ``bias`` FP32 ``[B, K <= 1024]`` (ids outside the vocabulary are ignored, the last of several
    for a token holds). ``mask`` int32 ``[B, N, ceil(V / 32)]``, bit ``v % 32`` of word ``v // 32``
    set where token ``v`` may follow. What is not given does not apply."""
    if logits.dim() not in (2, 3):
        raise ValueError("logits must be [B, V] or [B, N, V]")
    code = _dtype_code(logits)
    device, shape = logits.device, logits.shape
    batch, nodes, vocab = shape if len(shape) == 3 else (shape[0], 1, shape[1])
    logits = logits if logits.is_contiguous() else logits.contiguous()
    keep = []  # arrays that the call reads

    def array(t, name, dtype, dims):
        if t is None:
            return None
        keep.append(_array(t, name, dtype, dims, device))
        return keep[-1].data_ptr()

    i32, f32 = torch.int32, torch.float32
    d = _lib.LogitsDesc()
    if history is not None:
        if history.dim() != 2 or history_lengths is None:
            raise ValueError("history must be [B, L], with its lengths")
        d.history_capacity = history.shape[1]
        if history.shape[1]:
            d.history = array(history, "history", i32, (batch, history.shape[1]))
        d.history_lengths = array(history_lengths, "history_lengths", i32, (batch,))
        d.prompt_lengths = array(prompt_lengths, "prompt_lengths", i32, (batch,))
    d.repetition = array(repetition, "repetition", f32, (batch,))
    d.frequency = array(frequency, "frequency", f32, (batch,))
    d.presence = array(presence, "presence", f32, (batch,))
    d.temperature = array(temperature, "temperature", f32, (batch,))
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias_ids is not None and bias_ids.dim() == 2 and bias_ids.shape[1]:
        d.bias_count = bias_ids.shape[1]
        d.bias_ids = array(bias_ids, "bias_ids", i32, (batch, bias_ids.shape[1]))
        d.bias = array(bias, "bias", f32, (batch, bias_ids.shape[1]))
    elif bias_ids is not None and bias_ids.dim() != 2:
        raise ValueError("bias_ids must be [B, K]")
    if mask is not None:
        words = (vocab + 31) // 32
        d.mask = array(mask, "mask", i32, (batch, words) if len(shape) == 2 and mask.dim() == 2 else (batch, nodes, words))
    if (drafts is None) != (ancestors is None):
        raise ValueError("drafts and ancestors go together")
    if drafts is not None:
        d.drafts = array(drafts, "drafts", i32, (batch, nodes))
        d.ancestors = array(ancestors, "ancestors", torch.int64, (batch, nodes))
    if out is None:
        out = torch.empty_like(logits, dtype=f32)
    elif out.dtype != f32 or out.shape != shape or out.device != device or not out.is_contiguous():
        raise ValueError("out must be contiguous FP32 of the logits' shape")
    _lib.call_on(device, "qk_process_logits", ctypes.byref(d), logits.data_ptr(), code, batch, nodes, vocab, out.data_ptr())
    return out


__all__ = ["process_logits"]
