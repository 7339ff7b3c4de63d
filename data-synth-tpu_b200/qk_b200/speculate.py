"""Speculative decoding over the synthetic decoder stack and a pool of cache pages.

A step verifies a tree of up to ``nodes`` drafted tokens per sequence in one pass of the model
(the reference decodes one token per step, ``run.py:251``): node 0 is the sequence's newest
token, whose key and value are not in the cache yet, and the drafts hang below it.

* ``plan_step`` gives every node its page, cache slot, rotary position and ancestor word;
* per layer, the decoder's own operators around ``write_slots`` and ``tree_attention``;
* ``process_logits`` applies the sampling rules to every node's logits, each with the tokens of
  its own path counted, and ``checked_argmax`` chooses a token after every node;
* :func:`accept` keeps the longest path whose every token is the choice after its parent, and the
  choice after its last node is the step's extra token. The kept nodes' keys and values move to the
  front of the step's slots (``write_slots`` again: the same bytes at other slots).

Nothing waits for the host. Drafts come from a callable; :func:`lookup_drafts` is one that needs no
second model.
"""

import torch

from . import _lib
from .decoder import Fp8Projections, checked_argmax
from .fp8 import check_status
from .packed import linear_bf16, linear_workspace
from .paged import empty_pool, empty_tables, plan_step, tree_attention, write_slots
from .sampling import process_logits


def lookup_drafts(history, lengths, nodes):
    """``(tokens [B, nodes], parents None, counts [B])``: node 0 is the newest token of ``history``
    ``[B, L]`` (``lengths[b]`` of them), and the chain below it is what followed that token where it
    last stood before."""
    at = torch.arange(history.shape[1], device=history.device)
    last = (lengths.long() - 1).clamp(min=0)
    newest = torch.gather(history, 1, last[:, None])
    place = torch.where((history == newest) & (at < last[:, None]), at, -1).amax(1)
    index = (place[:, None] + torch.arange(nodes, device=history.device)).clamp(min=0)
    tokens = torch.gather(history, 1, index.clamp(max=history.shape[1] - 1))
    tokens[:, :1] = newest
    follow = torch.where(place >= 0, (last - place).clamp(max=nodes), 1)
    return tokens, None, follow.to(torch.int32)


def accept(tokens, parents, ancestors, counts, choices):
    """The path that a step keeps: ``(best [B], path [B, N], ranks [B, N], kept [B])``. ``choices``
    ``[B, N]`` is the token chosen after each node; node 0 is kept, and a node is where its parent is
    and its token is the choice after the parent. ``best`` is the deepest kept node (the first of
    several), ``path`` marks it and its ancestors, ``ranks`` their places on the path, ``kept`` their
    number. ``parents`` None: a chain; a parent that is not an earlier node counts as -1, as for
    :func:`~qk_b200.paged.plan_step`, and those of nodes past ``counts`` may be anything."""
    batch, nodes = tokens.shape
    node = torch.arange(nodes, device=tokens.device)
    up = (node - 1).expand(batch, nodes) if parents is None else parents.long()
    up = torch.where((up >= -1) & (up < node), up, -1)
    match = (tokens == torch.gather(choices, 1, up.clamp(min=0)).to(tokens.dtype)) & (up >= 0)
    match[:, 0] = True
    bits = (match.long() << node).sum(1, keepdim=True)
    live = (node < counts[:, None]) & ((ancestors & ~bits) == 0)
    depth = ((ancestors[:, :, None] >> node) & 1).sum(-1)
    best = torch.where(live, depth * nodes - node, -1).argmax(1)
    word = torch.gather(ancestors, 1, best[:, None])
    path = ((word >> node) & 1).bool() & (counts[:, None] > 0)
    ranks = path.long().cumsum(1) - 1
    return best, path, ranks, path.sum(1).to(torch.int32)


class SpeculativeGeneration:
    """``batch`` sequences of up to ``context`` tokens over ``model`` (a one-rank
    :class:`~qk_b200.decoder.SyntheticDecoder`), verified ``nodes`` drafted tokens at a time.
    ``rules``: keyword arguments of :func:`~qk_b200.sampling.process_logits` (``repetition``,
    ``frequency``, ``bias_ids``, ...). ``pages`` (default: enough for every sequence) sizes the pool."""

    def __init__(self, model, batch, context, nodes=8, page_size=64, vocab=151936, pages=None, drafts=lookup_drafts,
                 rules=None, seed=0):
        if model.world != 1:
            raise ValueError("speculative generation runs on one rank")
        if not 1 <= nodes <= 64:
            raise ValueError("a draft tree has 1 to 64 nodes")
        cfg, dev = model.cfg, model.device
        self.model, self.batch, self.context, self.nodes, self.page = model, batch, context, nodes, page_size
        self.drafts, self.rules = drafts, dict(rules or {})
        width = -(-(context + nodes) // page_size)
        self.table, self.held, self.ring, self.span = empty_tables(batch, width, pages or batch * width, dev)
        self.pools = [empty_pool(self.ring.shape[0], page_size, kv_heads=cfg.kv_heads, head_dim=cfg.head_dim, device=dev)
                      for _ in model.layers]
        g = torch.Generator(device=dev).manual_seed(seed + 3)
        self.embedding = (torch.randn((vocab, cfg.hidden), device=dev, generator=g) * 0.02).to(torch.bfloat16)
        self.final_norm = torch.ones(cfg.hidden, dtype=torch.bfloat16, device=dev)
        self.history = torch.zeros((batch, context + nodes + 1), dtype=torch.int32, device=dev)
        self.cached = torch.zeros(batch, dtype=torch.int32, device=dev)  # tokens in the cache
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)  # tokens of the history
        self.prompts = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.status = torch.zeros(batch, dtype=torch.int32, device=dev)  # of all plans so far
        rows, H, bf = batch * nodes, cfg.hidden, dict(dtype=torch.bfloat16, device=dev)
        hq, kv, hd = cfg.query_heads, cfg.kv_heads, cfg.head_dim
        self.h, self.a, self.y = (torch.empty((rows, H), **bf) for _ in range(3))
        self.qkv = torch.empty((rows, 2 * (hq + kv) * hd), **bf)
        self.q, self.gate = (torch.empty((batch, nodes, hq, hd), **bf) for _ in range(2))
        self.keys, self.values = ([torch.empty((batch, nodes, kv, hd), **bf) for _ in model.layers] for _ in range(2))
        self.router = torch.empty((rows, cfg.experts), dtype=torch.float32, device=dev)
        self.ids = torch.empty((rows, cfg.top_k + 1), dtype=torch.int32, device=dev)
        self.weights = torch.empty((rows, cfg.top_k + 1), **bf)
        self.linear_ws = {}
        self.fp8 = Fp8Projections(cfg, rows, dev) if cfg.dense == "fp8" else None
        self.moe_ws = torch.empty(max(int(_lib.load().qk_moe_workspace_bytes(model.desc, rows)), 16), dtype=torch.uint8,
                                  device=dev)

    def _linear(self, x, w, out):
        if x.shape[0] > 256:  # a library product beyond the decode batches of the tcgen05 pass
            return torch.matmul(x, w.t(), out=out)
        key = tuple(w.shape)
        if key not in self.linear_ws:
            self.linear_ws[key] = linear_workspace(x.shape[0], w.shape[1], w.shape[0], x.device)
        return linear_bf16(x, w, out=out, workspace=self.linear_ws[key])

    def forward(self, tokens, counts, parents=None):
        """``tokens`` ``[B, nodes]`` (the first ``counts[b]`` of each row) behind the cached ones of
        every sequence, in a tree of ``parents``: ``(hidden [B * nodes, H], plan)``. Padding may hold any
        id; a draft outside the vocabulary is embedded as the nearest one in it, and never accepted."""
        m, cfg, lib, P = self.model, self.model.cfg, _lib.load(), _lib.ptr
        rows, H = self.batch * self.nodes, cfg.hidden
        hq, kv, hd = cfg.query_heads, cfg.kv_heads, cfg.head_dim
        plan = plan_step(self.table, self.held, self.ring, self.span, self.cached, counts, nodes=self.nodes,
                         page_size=self.page, parents=parents)
        self.held, self.span = plan.held, plan.span
        self.status |= plan.status
        x = self.embedding.index_select(0, tokens.reshape(-1).long().clamp(0, self.embedding.shape[0] - 1))
        st = _lib.stream_handle(m.device)
        fp8, last = self.fp8, len(m.layers) - 1
        if fp8:  # as in the decode step: the attention norms leave as codes
            fp8.norm(x, None, m.layers[0].attn_norm, st)
        else:
            _lib.check(lib.qk_rms_norm(P(x), P(m.layers[0].attn_norm), rows, H, cfg.eps, P(self.h), st))
        for li, L in enumerate(m.layers):
            k, v = self.keys[li], self.values[li]
            if fp8:
                fp8.qkv(L.w_qkv, self.qkv, st)
            else:
                self._linear(self.h, L.w_qkv, self.qkv)
            _lib.check(lib.qk_qk_norm_rope(P(self.qkv), P(L.q_norm), P(L.k_norm), P(m.inv_freq), P(plan.positions), rows,
                                           hq, kv, hd, cfg.rotary_dim, cfg.eps, P(self.q), P(self.gate), P(k), P(v), st))
            write_slots(self.pools[li], k, v, plan.slots)
            o = tree_attention(self.q, self.pools[li], self.table, self.cached, plan.ancestors, page_size=self.page,
                               counts=counts, gate=self.gate)
            if fp8:
                fp8.out(o.view(rows, hq * hd), L.w_o, self.a, st)
            else:
                self._linear(o.view(rows, hq * hd), L.w_o, self.a)
            _lib.check(lib.qk_residual_rms_norm(P(x), P(self.a), P(L.ffn_norm), rows, H, cfg.eps, P(x), P(self.h), st))
            _lib.check(lib.qk_router_logits(P(self.h), P(L.router), rows, H, cfg.experts, P(self.router), st))
            _lib.check(lib.qk_router_select_shared(P(self.router), None, rows, cfg.experts, cfg.top_k, P(self.h),
                                                   P(L.shared_router), H, cfg.experts, 0, P(self.ids), P(self.weights), st))
            _lib.check(lib.qk_moe_forward(m.desc, P(L.experts["gate"]), P(L.experts["up"]), P(L.experts["down"]), P(self.h),
                                          P(self.ids), P(self.weights), rows, _lib.QK_OUT_BF16, P(self.y), P(self.moe_ws),
                                          self.moe_ws.numel(), st))
            if fp8 and li < last:
                fp8.norm(x, self.y, m.layers[li + 1].attn_norm, st)
                continue
            norm = m.layers[li + 1].attn_norm if li < last else self.final_norm
            _lib.check(lib.qk_residual_rms_norm(P(x), P(self.y), P(norm), rows, H, cfg.eps, P(x), P(self.h), st))
        return self.h, plan

    def logits(self, hidden, tokens, plan):
        """The processed logits ``[B, nodes, V]`` after every node. The history holds all tokens up to
        node 0, which is its last: the drafts below it count by their paths."""
        raw = torch.matmul(hidden, self.embedding.t()).view(self.batch, self.nodes, -1)
        drafts = tokens.clone()
        drafts[:, 0] = -1
        return process_logits(raw, history=self.history, history_lengths=self.lengths, prompt_lengths=self.prompts,
                              drafts=drafts, ancestors=plan.ancestors, **self.rules)

    def prefill(self, prompts):
        """``prompts``: token lists, one per sequence. All but the last token of each go into the cache,
        ``nodes`` at a time; the last is the first step's node 0. What was generated before is forgotten, and
        all pages are free again."""
        if len(prompts) != self.batch or any(not 0 < len(p) <= self.context for p in prompts):
            raise ValueError("one prompt of 1 to `context` tokens per sequence")
        if any(not 0 <= t < self.embedding.shape[0] for p in prompts for t in p):
            raise ValueError("a prompt's tokens must lie in the vocabulary")
        dev = self.model.device
        self.table, self.held, self.ring, self.span = empty_tables(self.batch, self.table.shape[1], self.ring.shape[0], dev)
        self.cached, self.status = torch.zeros_like(self.cached), torch.zeros_like(self.status)
        self.history.zero_()
        longest = max(len(p) for p in prompts)
        rows = torch.tensor([list(p) + [0] * (longest - len(p)) for p in prompts], dtype=torch.int32)
        self.history[:, :longest] = rows.to(dev)
        self.lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32).to(dev)
        self.prompts = self.lengths.clone()
        for first in range(0, longest - 1, self.nodes):
            counts = (self.lengths - 1 - first).clamp(0, self.nodes).to(torch.int32)
            self.forward(self.history[:, first:first + self.nodes].contiguous(), counts)
            self.cached = self.cached + counts

    def step(self):
        """One verify step; returns the number of new tokens per sequence (int32 ``[B]``, on the device).
        A sequence at its context's end stays as it is."""
        tokens, parents, counts = self.drafts(self.history, self.lengths, self.nodes)
        counts = torch.minimum(counts, self.context - self.cached).clamp(min=0).to(torch.int32)
        hidden, plan = self.forward(tokens, counts, parents)
        choices = checked_argmax(self.logits(hidden, tokens, plan).view(self.batch * self.nodes, -1))[:, 0]
        choices = choices.view(self.batch, self.nodes)
        best, path, ranks, kept = accept(tokens, parents, plan.ancestors, counts, choices)
        # the kept nodes' keys and values move to the front of the step's slots
        front = torch.gather(plan.slots, 1, ranks.clamp(min=0))
        move = torch.where(path & (front != plan.slots), front, -1)
        for li in range(len(self.pools)):
            write_slots(self.pools[li], self.keys[li], self.values[li], move)
        # node 0 is in the history; the path behind it and the choice after its end follow
        at = self.lengths[:, None].long() + torch.where(path, ranks - 1, 0)
        fresh = path & (ranks > 0)
        room = self.history.shape[1]
        grown = torch.cat([self.history, self.history[:, :1]], 1)
        grown.scatter_(1, torch.where(fresh, at.clamp(max=room - 1), room), tokens.to(torch.int32))
        end = torch.where(kept > 0, self.lengths + kept - 1, room).long()
        grown.scatter_(1, end[:, None], torch.gather(choices, 1, best[:, None]))
        self.history = grown[:, :room].contiguous()
        self.cached = self.cached + kept
        self.lengths = self.lengths + kept
        return kept

    def generate(self, steps):
        """``steps`` verify steps; returns the token lists so far (prompts included)."""
        for _ in range(steps):
            self.step()
        lengths = self.lengths.tolist()
        if bool(self.status.any()):
            raise RuntimeError(f"the pool of pages ran out or a draft was invalid: {self.status.tolist()}")
        tree_attention.check_status(self.model.device)
        if self.fp8:
            check_status(self.model.device)
        return [row[:n] for row, n in zip(self.history.tolist(), lengths)]


__all__ = ["SpeculativeGeneration", "accept", "lookup_drafts"]
