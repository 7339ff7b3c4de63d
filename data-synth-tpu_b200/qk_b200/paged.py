"""Paged Q8 cache and draft trees: the operators of one speculative-decoding (verify) step.

A pool of pages is a Q8 cache of the framework's layout (:func:`empty_pool`: one row whose time
axis is the pool; a static ``[B, T]`` cache serves as well, its pages numbered row by row).
Request ``b`` owns the pages of row ``b`` of the block table: its token ``t`` lives in slot
``table[b, t // page] * page + t % page``. One step of up to ``N`` drafted tokens per request::

    plan = plan_step(table, held, ring, span, lengths, counts, nodes=N, page_size=P, parents=parents)
    held, span = plan.held, plan.span
    for each layer:
        write_slots(cache, k, v, plan.slots)                       # k, v [B, N, kv, hd]
        o = tree_attention(q, cache, table, lengths, plan.ancestors, page_size=P, counts=counts)

Drafts form a tree: ``parents[b, i]`` is the node above node ``i`` (an earlier one, or -1 for the
prefix itself), without parents they form a chain. With ``N = 1`` the step is plain decoding.
The reference has no counterpart (a static cache, one token per step).
"""

from typing import NamedTuple

import torch

from . import _lib
from .attention_cache import _dtype_code


def empty_pool(pages, page_size, *, kv_heads=2, head_dim=256, device=None):
    """A Q8 cache of one row and ``pages * page_size`` slots, zeroed: ``k`` / ``v`` int8
    ``[1, slots, kv * hd]``, ``k_scale`` / ``v_scale`` BF16 ``[G, slots]``."""
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two in [16, 1024]")
    if pages < 1 or pages * page_size > 0x7FFFFFFF:
        raise ValueError("the pool's slots must fit 31 bits")
    if head_dim % min(32, head_dim):
        raise ValueError("KV head dimension must divide into cache quantization groups")
    device = torch.device(device or "cuda")
    slots, groups = pages * page_size, kv_heads * (head_dim // min(32, head_dim))
    cache = {n: torch.zeros((1, slots, kv_heads * head_dim), dtype=torch.int8, device=device) for n in ("k", "v")}
    cache.update({n: torch.zeros((groups, slots), dtype=torch.bfloat16, device=device)
                  for n in ("k_scale", "v_scale")})
    return cache


def empty_tables(batch, width, pages, device=None):
    """``(table, held, ring, span)`` of ``batch`` requests that hold no page, all ``pages`` free."""
    device = torch.device(device or "cuda")
    return (torch.full((batch, width), -1, dtype=torch.int32, device=device),
            torch.zeros(batch, dtype=torch.int32, device=device),
            torch.arange(pages, dtype=torch.int32, device=device),
            torch.tensor([0, pages], dtype=torch.int32, device=device))


class StepPlan(NamedTuple):
    slots: torch.Tensor      # int32 [B, N], -1: no slot
    positions: torch.Tensor  # int32 [B, N]
    ancestors: torch.Tensor  # int64 [B, N], bit j: node j is the node or above it (None: N > 64)
    held: torch.Tensor       # int32 [B]: pages held after the step
    span: torch.Tensor       # int32 [2]: the ring's head and number of free pages after it
    status: torch.Tensor     # int32 [B]: 0, or the sum of NO_PAGES, TABLE_FULL, BAD_LENGTH, BAD_PARENT


NO_PAGES, TABLE_FULL, BAD_LENGTH, BAD_PARENT = 1, 2, 4, 8


def _array(t, name, dtype, shape, device):
    """``t`` on ``device``, contiguous and of the dtype; a ValueError for another shape."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype or t.device != device:
        t = t.to(device=device, dtype=dtype)
    return t if t.is_contiguous() else t.contiguous()


def _in_place(t, name, dims):
    if t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous() or not t.is_cuda:
        raise TypeError(f"{name} must be a contiguous int32 CUDA tensor of {dims} dimension(s): it is updated in place")


def plan_step(table, held, ring, span, lengths, counts, *, nodes, page_size, parents=None, out=None):
    """Pages, cache slots, positions and ancestor words of the next ``counts[b] <= nodes`` tokens
    after ``lengths[b]``. ``table`` ``[B, width]`` and ``ring`` ``[pages]`` (int32) change in
    place; the pages ``held`` and the ring's ``span`` after the step come back in the plan, whose
    arrays may be a former plan's (``out``, for steps in a CUDA graph; not the one whose ``held``
    and ``span`` come in). Requests give back pages they need no more (``lengths[b] = counts[b]
    = 0`` ends one). A request that finds no pages keeps what it holds, gets slot -1 beyond them
    and ``NO_PAGES`` in ``status``."""
    _in_place(table, "table", 2)
    _in_place(ring, "ring", 1)
    device = table.device
    if ring.device != device:
        raise ValueError("table and ring must be on one device")
    batch, width = table.shape
    i32 = torch.int32
    held = _array(held, "held", i32, (batch,), device)
    span = _array(span, "span", i32, (2,), device)
    lengths = _array(lengths, "lengths", i32, (batch,), device)
    counts = _array(counts, "counts", i32, (batch,), device)
    if nodes < 1:
        raise ValueError("nodes must be positive")
    if parents is not None:
        if nodes > 64:
            raise ValueError("a draft tree has at most 64 nodes")
        parents = _array(parents, "parents", i32, (batch, nodes), device)
    if out is None:
        slots = torch.empty((batch, nodes), dtype=i32, device=device) if parents is None else torch.empty_like(parents)
        out = StepPlan(slots, torch.empty_like(slots),
                       torch.empty((batch, nodes), dtype=torch.int64, device=device) if nodes <= 64 else None,
                       torch.empty_like(held), torch.empty_like(span), torch.empty_like(held))
    elif out.slots.shape != (batch, nodes) or out.slots.device != device:
        raise ValueError("out must be the plan of as many requests and nodes on the same device")
    _lib.call_on(device, "qk_paged_plan", table.data_ptr(), held.data_ptr(), ring.data_ptr(), span.data_ptr(),
                 lengths.data_ptr(), counts.data_ptr(), None if parents is None else parents.data_ptr(), batch, width,
                 ring.shape[0], page_size, nodes, out.slots.data_ptr(), out.positions.data_ptr(),
                 None if out.ancestors is None else out.ancestors.data_ptr(), out.held.data_ptr(), out.span.data_ptr(),
                 out.status.data_ptr())
    return out


def _cache_geometry(cache, kv, hd, device):
    """``(k, v, k_scale, v_scale, rows, T)`` of a Q8 cache on ``device``, whose arrays must be of the
    framework's layout."""
    k, v, ks, vs = cache["k"], cache["v"], cache["k_scale"], cache["v_scale"]
    shape, plane = k.shape, ks.shape
    if len(shape) != 3 or shape[2] != kv * hd or plane != (shape[0] * (kv * hd // min(32, hd)), shape[1]):
        raise ValueError("cache must hold codes [R, T, kv * hd] and scale planes [R * G, T] of these heads")
    if k.dtype != torch.int8 or v.dtype != torch.int8 or ks.dtype != torch.bfloat16 or vs.dtype != torch.bfloat16:
        raise TypeError("cache codes must be int8 and scales BF16")
    if not (k.device == v.device == ks.device == vs.device == device):
        raise ValueError("the cache must be on the device of the tokens")
    if v.shape != shape or vs.shape != plane or not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous()
                                                     and vs.is_contiguous()):
        raise ValueError("cache keys and values must be contiguous and of the same shape")
    return k, v, ks, vs, shape[0], shape[1]


def _tokens(x, width):
    """``x`` ``[..., kv, hd]`` as rows of ``width`` values: ``(x, stride)``; copied only where its
    tokens are not evenly spaced 16-byte aligned rows."""
    if x.data_ptr() % 16:  # a contiguous tensor is itself its contiguous(): only a copy moves it
        return x.clone(memory_format=torch.contiguous_format), width
    if x.is_contiguous():
        return x, width
    per = 16 // x.element_size()
    lead = x.shape[:-2]
    dense = x.stride(-1) == 1 and (x.shape[-2] == 1 or x.stride(-2) == x.shape[-1])
    step = x.stride(-3) if lead else width
    for i in range(len(lead) - 1):
        dense = dense and (lead[i] == 1 or x.stride(i) == step * _count(lead[i + 1:]))
    if not dense or step < width or step % per:
        return x.contiguous(), width
    return x, step


def _count(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def write_slots(cache, key, value, slots):
    """Quantise ``key`` / ``value`` ``[..., kv, hd]`` (BF16 or FP32, any even token stride) into the
    cache slots ``slots`` ``[...]``, in place; slots outside the cache (-1: padding) are dropped, and
    no two tokens may name one slot. The codec of :func:`~qk_b200.attention_cache.write_quantized`."""
    if key.shape != value.shape or key.dim() < 2 or key.shape[:-2] != slots.shape:
        raise ValueError("key and value must be [..., kv, hd] with one slot for every token")
    kv, hd = key.shape[-2:]
    device = key.device
    k, v, ks, vs, rows, time = _cache_geometry(cache, kv, hd, device)
    code = _dtype_code(key)
    if value.dtype != key.dtype or value.device != device:
        value = value.to(device=device, dtype=key.dtype)
    key, key_stride = _tokens(key, kv * hd)
    value, value_stride = _tokens(value, kv * hd)
    slots = _array(slots, "slots", torch.int32, slots.shape, device)
    _lib.call_on(device, "qk_kv_q8_write_slots", key.data_ptr(), value.data_ptr(), code, key_stride, value_stride,
                 slots.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), slots.numel(), rows, time, kv,
                 hd)
    return cache


class TreeAttention:
    """Attention of drafted tokens over a paged Q8 cache, with a workspace per stream; calls in a graph have
    theirs in the graph's memory, so that graphs may be replayed beside one another."""

    def __init__(self):
        self._ws = {}
        self._need = {}

    def _workspace(self, device, geometry):
        """The workspace of a call on the device's current stream, of the size for ``(B, N, hq, kv, hd)``."""
        need = self._need.get(geometry)
        if need is None:
            with torch.cuda.device(device):
                need = self._need[geometry] = int(_lib.load().qk_tree_attention_workspace_bytes(*geometry))
        if torch.cuda.current_device() == device.index:
            capturing = torch._C._cuda_isCurrentStreamCapturing()
        else:
            with torch.cuda.device(device):
                capturing = torch._C._cuda_isCurrentStreamCapturing()
        if capturing:
            return torch.empty(need, dtype=torch.uint8, device=device)
        key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
        ws = self._ws.get(key)
        if ws is None or ws.numel() < need:
            ws = self._ws[key] = torch.zeros(need, dtype=torch.uint8, device=device)
        return ws

    def __call__(self, q, cache, table, lengths, ancestors, *, page_size, counts=None, gate=None, scale=None, out=None):
        """``q`` BF16 ``[B, N, hq, hd]`` (``N <= 64``; tokens may be strided) of nodes whose keys and
        values are already in the cache as tokens ``lengths[b] + i``: each sees the prefix
        ``t < lengths[b]`` and the nodes of its word of ``ancestors`` (int64 ``[B, N]``,
        :func:`plan_step`); ``scale`` defaults to ``hd ** -0.5``. Returns BF16 ``[B, N, hq, hd]``,
        times ``sigmoid(gate)`` where a gate is given; nodes past ``counts[b]`` are zero. Queries must
        stay within 2^22 and keys within 2^20; a node that sees a draft that is not finite is NaN."""
        if q.dtype != torch.bfloat16 or q.dim() != 4:
            raise TypeError("q must be BF16 [B, N, query_heads, head_dim]")
        shape, device = q.shape, q.device
        batch, nodes, hq, hd = shape
        if hd not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if not 1 <= nodes <= 64:
            raise ValueError("a request has 1 to 64 nodes")
        if not q.is_cuda:
            raise ValueError("expected CUDA tensors")
        kv = cache["k"].shape[-1] // hd
        if kv < 1 or hq % kv:
            raise ValueError("Head counts must have integer repetition factors")
        k, v, ks, vs, rows, time = _cache_geometry(cache, kv, hd, device)
        if table.dim() != 2 or table.shape[0] != batch:
            raise ValueError("table must be [B, width]")
        q, stride = _tokens(q, hq * hd)
        table = _array(table, "table", torch.int32, table.shape, device)
        lengths = _array(lengths, "lengths", torch.int32, (batch,), device)
        ancestors = _array(ancestors, "ancestors", torch.int64, (batch, nodes), device)
        if counts is not None:
            counts = _array(counts, "counts", torch.int32, (batch,), device)
        if gate is not None:
            gate = _array(gate, "gate", torch.bfloat16, shape, device)
            if gate.data_ptr() % 16:
                gate = gate.clone()
        if out is None:
            out = torch.empty(shape, dtype=torch.bfloat16, device=device) if stride != hq * hd else torch.empty_like(q)
        elif out.dtype != torch.bfloat16 or out.shape != shape or out.device != device or not out.is_contiguous():
            raise ValueError("out must be contiguous BF16 of q's shape")
        elif out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
            q, stride = q.clone(memory_format=torch.contiguous_format), hq * hd  # read until the last output is written
        ws = self._workspace(device, (batch, nodes, hq, kv, hd))
        _lib.call_on(device, "qk_tree_attention", q.data_ptr(), stride, k.data_ptr(), v.data_ptr(), ks.data_ptr(),
                     vs.data_ptr(), table.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr(),
                     ancestors.data_ptr(), None if gate is None else gate.data_ptr(), hd ** -0.5 if scale is None else scale,
                     batch, nodes, hq, kv, hd, rows, time, table.shape[1], page_size, out.data_ptr(), ws.data_ptr(),
                     ws.numel())
        return out

    def check_status(self, device=None):
        """Raise what earlier calls on the device reported, in graphs and on other streams too as far as they have
        run (a table entry outside the cache, a length outside the table, a bounded wait that gave up);
        synchronises the current stream."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        _lib.call_on(device, "qk_tree_attention_check", None)


tree_attention = TreeAttention()


__all__ = ["BAD_LENGTH", "BAD_PARENT", "NO_PAGES", "TABLE_FULL", "StepPlan", "TreeAttention", "empty_pool",
           "empty_tables", "plan_step", "tree_attention", "write_slots"]
