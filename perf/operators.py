"""What is measured of the speculative-decoding operators: one verify step over a paged Q8 cache.

A verify step plans the pages and cache slots of every request's drafted tokens (``plan``),
quantises their keys and values into the paged Q8 cache (``write``), attends from every
drafted token to its request's prefix and to its own ancestors in the draft tree
(``attention``) and turns the head's logits into the ones to choose from, with penalties for
repeated tokens, biases and grammar masks (``logits``).

With ``own`` false, ``run`` computes each operator in its plain form (elementary torch
operations in 32 bits, rounded once at the end); with ``own`` true it calls ``qk_b200``.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_GROUP = 32  # channels per scale of the Q8 cache


def listed():
    return [
        # one decode step of a large batch: a slot for every request, a few new pages
        dict(name="plan decode b64", op="plan", batch=64, nodes=1, context=8192, page=256, tree=False),
        # a tree of drafts for every request of a full server, small pages
        dict(name="plan tree b256 n64", op="plan", batch=256, nodes=64, context=32768, page=16, tree=True),
        # a prompt chunk of every request: long slot maps without a tree
        dict(name="plan prompt b61 n2048", op="plan", batch=61, nodes=2048, context=4099, page=64, tree=False),
        # one new token for each of 64 requests, BF16 keys and values
        dict(name="write decode b64", op="write", tokens=64, slots=1024, page=256, kv=2, hd=256, dtype="bf16"),
        # a ragged prompt chunk, FP32 keys and values, 8 heads of 128
        dict(name="write prompt 8111", op="write", tokens=8111, slots=8448, page=64, kv=8, hd=128, dtype="f32"),
        # the single-token form: plain decoding of one sequence, where latency counts
        dict(name="attention b1 n1 c4096", op="attention", batch=1, nodes=1, context=4096, page=256, hq=16, kv=2,
             hd=256, gate=True),
        # a tree of 16 for one long sequence: the cache read split over the whole GPU
        dict(name="attention b1 n16 c32768", op="attention", batch=1, nodes=16, context=32768, page=256, hq=16, kv=2,
             hd=256, gate=True),
        # a serving batch with small trees and ragged lengths
        dict(name="attention b32 n8 c8192", op="attention", batch=32, nodes=8, context=8192, page=256, hq=16, kv=2,
             hd=256, gate=True),
        # odd sizes, small pages, three query heads per KV head of 128
        dict(name="attention b5 n13 c3001 hd128", op="attention", batch=5, nodes=13, context=3001, page=16, hq=24,
             kv=8, hd=128, gate=False),
        # the widest trees: 512 query rows per KV head, bound by the tensor cores
        dict(name="attention b16 n64 c16384", op="attention", batch=16, nodes=64, context=16384, page=64, hq=16, kv=2,
             hd=256, gate=True),
        # sampling for one sequence: latency
        dict(name="logits b1", op="logits", batch=1, nodes=1, vocab=151936, history=2048, dtype="bf16", mask=True),
        # every node of 16 trees, a vocabulary that no vector divides, long histories
        dict(name="logits b16 n24 odd", op="logits", batch=16, nodes=24, vocab=151937, history=16384, dtype="f32",
             mask=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attention", "attention", "attention", "logits", "logits"])
    if op == "plan":
        tree = rng.random() < 0.5
        nodes = _log_int(rng, 1, 64 if tree else 2048)
        batch = min(_log_int(rng, 1, 256), max(1, 61 * 2048 // nodes))
        return dict(op=op, batch=batch, nodes=nodes, context=_log_int(rng, 1, 32768), page=rng.choice([16, 32, 64, 128, 256]),
                    tree=tree)
    if op == "write":
        kv, hd = rng.choice([(2, 256), (8, 128), (4, 64), (1, 256), (3, 128)])
        tokens = _log_int(rng, 1, 8111)
        page = rng.choice([16, 64, 256])
        return dict(op=op, tokens=tokens, slots=(tokens + 300 + page - 1) // page * page, page=page, kv=kv, hd=hd,
                    dtype=rng.choice(["bf16", "f32"]))
    if op == "attention":
        hq, kv, hd = rng.choice([(16, 2, 256), (24, 2, 256), (24, 8, 128), (32, 8, 128), (4, 4, 64), (16, 2, 256)])
        batch, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 64)
        context = _log_int(rng, 1, 32768)
        while batch * nodes * hq * context * hd > 16 * 64 * 16 * 16384 * 256 or batch * context * kv * hd > 16 * 16384 * 512:
            context = context * 2 // 3
        return dict(op=op, batch=batch, nodes=nodes, context=max(context, 1), page=rng.choice([16, 32, 64, 128, 256]),
                    hq=hq, kv=kv, hd=hd, gate=rng.random() < 0.5)
    vocab = rng.choice([151936, 151937, _log_int(rng, 1000, 151936)])
    batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 24)
    nodes = max(1, min(nodes, 16 * 24 // batch))
    return dict(op=op, batch=batch, nodes=nodes, vocab=vocab, history=_log_int(rng, 1, 16384),
                dtype=rng.choice(["bf16", "f32"]), mask=rng.random() < 0.7)


# ---- inputs ------------------------------------------------------------------------------


def _device():
    return torch.device("cuda")


def _ints(g, low, high, shape):
    return torch.randint(low, high, shape, generator=g, device=g.device, dtype=torch.int32)


def _requests(g, batch, context, nodes):
    """Ragged prefix lengths in [1, context] (the first the longest; of four or more requests
    the second is empty) and draft counts in [1, nodes] (of four or more the third has none)."""
    lengths = _ints(g, 1, context + 1, (batch,))
    counts = _ints(g, (nodes + 1) // 2, nodes + 1, (batch,)).clamp_(min=1)
    lengths[0] = context
    counts[0] = nodes
    if batch >= 4:
        lengths[1] = 0
        counts[2] = 0
    return lengths, counts


def _parents(g, batch, nodes):
    """Draft trees: half of the nodes continue the node before them, the others hang on a
    random earlier node or start a branch of their own (-1)."""
    i = torch.arange(nodes, device=g.device)
    u = torch.rand((batch, nodes), generator=g, device=g.device)
    chain = torch.rand((batch, nodes), generator=g, device=g.device) < 0.5
    other = (u * (i + 1)).long() - 1
    return torch.where(chain, (i - 1).expand(batch, nodes), other).to(torch.int32)


def _ancestor_matrix(parents):
    """[B, N, N]: whether node j is node i or one of its ancestors."""
    nodes = parents.shape[1]
    j = torch.arange(nodes, device=parents.device)
    step = (parents[:, :, None] == j).float() + (j[:, None] == j)
    return torch.linalg.matrix_power(step, 64) > 0.5


def _bits(matrix):
    """[B, N, N] truth values -> int64 words, bit j of word i from entry (i, j)."""
    j = torch.arange(matrix.shape[2], device=matrix.device)
    return torch.bitwise_left_shift(matrix.long(), j).sum(-1)


def _cache(g, slots, kv, hd):
    """A Q8 cache of one row whose keys and values are N(0, 1)."""
    cache = {}
    width, groups = kv * hd, kv * hd // _GROUP
    for name in ("k", "v"):
        x = torch.randn((slots, groups, _GROUP), generator=g, device=g.device)
        scale = (x.abs().amax(-1, keepdim=True) / 127).to(torch.bfloat16)
        cache[name] = (x / scale.float()).round_().clamp_(-127, 127).to(torch.int8).view(1, slots, width)
        cache[name + "_scale"] = scale.view(slots, groups).t().contiguous()
        del x
    return cache


def prepare(case, seed):
    g = torch.Generator(device=_device()).manual_seed(seed)
    op, dev = case["op"], _device()
    if op == "plan":
        batch, nodes, page = case["batch"], case["nodes"], case["page"]
        lengths, counts = _requests(g, batch, case["context"], nodes)
        width = (case["context"] + nodes + page - 1) // page + 1
        # the pages of the prefix are held, some requests hold a spare page of rejected drafts
        held = (lengths + page - 1) // page + (_ints(g, 0, 4, (batch,)) == 0)
        order = torch.randperm(batch * width, generator=g, device=dev).to(torch.int32)
        column = torch.arange(width, device=dev)
        table = torch.where(column < held[:, None], order.view(batch, width), -1).to(torch.int32)
        # the free pages wait in a ring that starts somewhere in the array
        free = torch.where(column < held[:, None], -1, order.view(batch, width)).flatten()
        free = free[torch.sort((free < 0).to(torch.int32), stable=True).indices]
        head = int(seed * 7919 % (batch * width))
        count = (free >= 0).sum().to(torch.int32)
        span = torch.stack([torch.tensor(head, dtype=torch.int32, device=dev), count])
        parents = _parents(g, batch, nodes) if case["tree"] else None
        return dict(op=op, page=page, nodes=nodes, lengths=lengths, counts=counts, held=held.to(torch.int32),
                    table=table, ring=torch.roll(free, head).contiguous(), span=span, parents=parents)
    if op == "write":
        tokens, kv, hd = case["tokens"], case["kv"], case["hd"]
        cache = _cache(g, case["slots"], kv, hd)
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        key = torch.randn((tokens, kv, hd), generator=g, device=dev).to(dtype)
        value = torch.randn((tokens, kv, hd), generator=g, device=dev).to(dtype)
        value[0, 0] = 0  # a group of zeros has the scale zero
        # one token in 16 is padding
        slots = torch.randperm(case["slots"], generator=g, device=dev)[:tokens].to(torch.int32)
        slots = torch.where(_ints(g, 0, 16, (tokens,)) == 0, -1, slots)
        every = torch.arange(case["slots"], dtype=torch.int32, device=dev)[None]
        return dict(op=op, cache=cache, key=key, value=value, slots=slots, every=every)
    if op == "attention":
        batch, nodes, page, hq, kv, hd = (case[n] for n in ("batch", "nodes", "page", "hq", "kv", "hd"))
        lengths, counts = _requests(g, batch, case["context"], nodes)
        width = (case["context"] + nodes + page - 1) // page
        table = torch.randperm(batch * width, generator=g, device=dev).to(torch.int32).view(batch, width)
        cache = _cache(g, batch * width * page, kv, hd)
        # normed and rotated queries; their norm's weight makes the scores somewhat peaked
        q = (torch.randn((batch, nodes, hq, hd), generator=g, device=dev) * 1.5).to(torch.bfloat16)
        gate = torch.randn((batch, nodes, hq, hd), generator=g, device=dev).to(torch.bfloat16) if case["gate"] else None
        ancestors = _bits(_ancestor_matrix(_parents(g, batch, nodes)))
        return dict(op=op, page=page, span=case["context"] + nodes, cache=cache, q=q, gate=gate, table=table,
                    lengths=lengths, counts=counts, ancestors=ancestors)
    batch, nodes, vocab, room = case["batch"], case["nodes"], case["vocab"], case["history"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = (torch.randn((batch, nodes, vocab), generator=g, device=dev) * 3).to(dtype)

    def tokens(shape):  # few tokens are frequent, most are rare
        return (torch.rand(shape, generator=g, device=dev) ** 4 * vocab).to(torch.int32).clamp_(max=vocab - 1)

    history_lengths = _ints(g, 0, room + 1, (batch,))
    history_lengths[0] = room
    uniform = lambda low, high: torch.rand((batch,), generator=g, device=dev) * (high - low) + low  # noqa: E731
    bias_ids = (torch.arange(64, device=dev) * 7919 + _ints(g, 0, vocab, (batch, 1))) % vocab
    bias_ids = torch.where(_ints(g, 0, 4, (batch, 64)) == 0, -1, bias_ids.to(torch.int32))
    if vocab % 7919 == 0 or vocab < 64:
        bias_ids = torch.arange(64, dtype=torch.int32, device=dev).expand(batch, 64).contiguous()
    mask = None
    if case["mask"]:
        mask = torch.randint(-2 ** 31, 2 ** 31, (batch, nodes, (vocab + 31) // 32), generator=g, device=dev).to(torch.int32)
        mask[-1, -1] = 0  # a grammar with no way on
        mask[0, 0] = -1   # and one that allows everything
    return dict(op=op, logits=logits, history=tokens((batch, room)), history_lengths=history_lengths,
                prompt_lengths=history_lengths // 2, repetition=uniform(1.0, 1.3), frequency=uniform(0.0, 0.5),
                presence=uniform(0.0, 0.5), temperature=uniform(0.5, 1.5), bias_ids=bias_ids,
                bias=torch.randn((batch, 64), generator=g, device=dev) * 4, mask=mask, drafts=tokens((batch, nodes)),
                ancestors=_bits(_ancestor_matrix(_parents(g, batch, nodes))))


# ---- the framework's operators -------------------------------------------------------------


def _package():
    folder = str(Path(__file__).resolve().parents[1] / "data-synth-tpu_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)


def _run_own(s):
    _package()
    if s["op"] == "plan":
        from qk_b200.paged import plan_step

        p = plan_step(s["table"], s["held"], s["ring"], s["span"], s["lengths"], s["counts"], nodes=s["nodes"],
                      page_size=s["page"], parents=s["parents"])
        return [p.slots, p.positions, p.held, p.span, p.status, s["table"], s["ring"],
                p.ancestors if s["parents"] is not None else p.slots]
    if s["op"] == "write":
        from qk_b200.attention_cache import CacheConfig, read_quantized
        from qk_b200.paged import write_slots

        cache = write_slots(s["cache"], s["key"], s["value"], s["slots"])
        c = CacheConfig(kv_heads=s["key"].shape[1], head_dim=s["key"].shape[2], query_heads=s["key"].shape[1])
        return [read_quantized(cache, name, s["every"], c, torch.bfloat16) for name in ("k", "v")]
    if s["op"] == "attention":
        from qk_b200.paged import tree_attention

        return tree_attention(s["q"], s["cache"], s["table"], s["lengths"], s["ancestors"], page_size=s["page"],
                              counts=s["counts"], gate=s["gate"])
    from qk_b200.sampling import process_logits

    return process_logits(s["logits"], history=s["history"], history_lengths=s["history_lengths"],
                          prompt_lengths=s["prompt_lengths"], repetition=s["repetition"], frequency=s["frequency"],
                          presence=s["presence"], temperature=s["temperature"], bias_ids=s["bias_ids"],
                          bias=s["bias"], mask=s["mask"], drafts=s["drafts"], ancestors=s["ancestors"])


# ---- the plain forms -----------------------------------------------------------------------


def _plan(s):
    table, held, ring, span, page, nodes = s["table"], s["held"], s["ring"], s["span"], s["page"], s["nodes"]
    width, pages = table.shape[1], ring.shape[0]
    lengths, counts = s["lengths"], s["counts"]
    head, count = span[0].long(), span[1]
    need = (lengths + counts + page - 1) // page
    want = (need - held).clamp(min=0)
    upto = torch.cumsum(want, 0)
    fits = ((upto <= count) & (need <= width)) | (want == 0)
    grow = torch.where(fits, want, 0)
    drop = (held - need).clamp(min=0)
    column = torch.arange(width, device=table.device)
    place = (upto - want)[:, None] + column - held[:, None]
    fresh = ring[(head + place) % pages]
    new = (column >= held[:, None]) & (column < (held + grow)[:, None])
    entries = torch.where(new, fresh, table)
    gone = (column >= need[:, None]) & (column < held[:, None])
    back = (torch.cumsum(drop, 0) - drop)[:, None] + column - need[:, None]
    to = torch.where(gone, (head + count + back) % pages, pages)
    longer = torch.cat([ring, ring[:1]])
    longer.scatter_(0, to.flatten(), table.flatten())
    ring.copy_(longer[:pages])
    table.copy_(entries)
    held_out = (held + grow - drop).to(torch.int32)
    span_out = torch.stack([((head + grow.sum()) % pages).to(torch.int32),
                            (count - grow.sum() + drop.sum()).to(torch.int32)])
    node = torch.arange(nodes, device=table.device)
    live = node < counts[:, None]
    at = lengths[:, None] + node
    have = live & (at // page < held_out[:, None])
    slots = torch.gather(entries, 1, (at // page).clamp(max=width - 1)) * page + at % page
    slots = torch.where(have, slots, -1).to(torch.int32)
    status = torch.where(fits, 0, torch.where(need <= width, 1, 2)).to(torch.int32)
    depth, ancestors = node, slots
    if s["parents"] is not None:
        seen = _ancestor_matrix(s["parents"]) & live[:, :, None] & live[:, None, :]
        depth = seen.sum(-1) - 1
        ancestors = _bits(seen)
    positions = torch.where(live, lengths[:, None] + depth, 0).to(torch.int32)
    return [slots, positions, held_out, span_out, status, table, ring, ancestors]


def _values(cache, name, dtype=torch.float32):
    """The values of a whole cache of one row, [1, slots, kv * hd]."""
    codes, scale = cache[name], cache[name + "_scale"]
    x = codes.to(dtype).view(codes.shape[1], -1, _GROUP) * scale.t()[:, :, None].to(dtype)
    return x.view(codes.shape)


def _write(s):
    cache, slots = s["cache"], s["slots"].long()
    room = cache["k"].shape[1]
    keep = torch.where(slots < 0, room, slots)  # padding goes to a slot past the end
    out = []
    for name, x in (("k", s["key"]), ("v", s["value"])):
        x = x.float().view(slots.shape[0], -1, _GROUP)
        scale = (x.abs().amax(-1) / 127).to(torch.bfloat16)
        divisor = torch.where(scale == 0, 1.0, scale.float())[..., None]
        codes = (x / divisor).round().clamp(-127, 127).to(torch.int8).view(slots.shape[0], -1)
        grown = torch.cat([cache[name][0], codes[:1]])
        grown[keep] = codes
        plane = torch.cat([cache[name + "_scale"], scale[:1].t()], 1)
        plane[:, keep] = scale.t()
        cache[name].copy_(grown[None, :room])
        cache[name + "_scale"].copy_(plane[:, :room])
        kv, hd = s["key"].shape[1:]
        out.append(_values(cache, name).to(torch.bfloat16).view(1, room, kv, hd))
    return out


def _attention(s):
    q, table, page, span = s["q"], s["table"], s["page"], s["span"]
    batch, nodes, hq, hd = q.shape
    kv = s["cache"]["k"].shape[2] // hd
    at = torch.arange(span, device=q.device)
    slots = table[:, at // page].long() * page + at % page
    keys, values = [], []
    for name, to in (("k", keys), ("v", values)):
        codes = s["cache"][name][0][slots].float().view(batch, span, -1, _GROUP)
        scale = s["cache"][name + "_scale"].t()[slots].float()
        to.append((codes * scale[..., None]).view(batch, span, kv, hd).transpose(1, 2))
    rows = q.float().view(batch, nodes, kv, hq // kv, hd).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, hd)
    scores = torch.matmul(rows, keys[0].transpose(2, 3)) * hd ** -0.5
    lengths, counts = s["lengths"][:, None, None], s["counts"][:, None, None]
    node = (at - lengths).clamp(0, 63)
    drafted = (at >= lengths) & (at < lengths + counts)
    seen = (at < lengths) | (drafted & ((s["ancestors"][:, :, None] >> node) & 1).bool())
    seen = seen & (torch.arange(nodes, device=q.device)[:, None] < counts)
    seen = seen[:, None, :, None, :]  # [B, kv, N, heads, span]
    scores = scores.view(batch, kv, nodes, hq // kv, span)
    top = torch.where(seen, scores, -1e30).amax(-1, keepdim=True)
    weights = torch.where(seen, torch.exp(scores - top), 0.0)
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, 1.0)
    out = torch.matmul(weights.view(batch, kv, -1, span), values[0]).view(batch, kv, nodes, hq // kv, hd)
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, nodes, hq, hd)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return out.to(torch.bfloat16)


def _logits(s, dtype=torch.float32):
    x = s["logits"].to(dtype)
    batch, nodes, vocab = x.shape
    room = s["history"].shape[1]
    at = torch.arange(room, device=x.device)
    valid = at < s["history_lengths"][:, None]
    said = valid & (at >= s["prompt_lengths"][:, None])
    ids = s["history"].long()
    count = torch.zeros((batch, vocab), dtype=dtype, device=x.device)
    context = count.clone().scatter_add_(1, ids, valid.to(dtype))
    count.scatter_add_(1, ids, said.to(dtype))
    # a drafted token counts in the rows of the nodes below it and in its own
    j = torch.arange(nodes, device=x.device)
    seen = ((s["ancestors"][:, :, None] >> j) & 1).to(dtype)
    drafted = torch.zeros_like(x).scatter_add_(2, s["drafts"].long()[:, None].expand(batch, nodes, nodes), seen)
    count = count[:, None] + drafted
    context = context[:, None] + drafted
    by = {n: s[n].to(dtype)[:, None, None] for n in ("repetition", "frequency", "presence", "temperature")}
    x = torch.where(context > 0, torch.where(x > 0, x / by["repetition"], x * by["repetition"]), x)
    x = x - by["frequency"] * count - by["presence"] * (count > 0)
    bias = torch.zeros((batch, vocab + 1), dtype=dtype, device=x.device)
    ids = torch.where((s["bias_ids"] >= 0) & (s["bias_ids"] < vocab), s["bias_ids"], vocab).long()
    bias.scatter_(1, ids, s["bias"].to(dtype))
    x = (x + bias[:, None, :vocab]) / by["temperature"]
    if s["mask"] is not None:
        v = torch.arange(vocab, device=x.device)
        x = torch.where(((s["mask"][:, :, v // 32] >> (v % 32)) & 1).bool(), x, -math.inf)
    return x


_PLAIN = {"plan": _plan, "write": _write, "attention": _attention, "logits": _logits}


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "plan":
        batch, nodes, page = case["batch"], case["nodes"], case["page"]
        # in: length, count, held pages, parents, a table entry per page of the new tokens; out:
        # slot, position (and a 64-bit ancestor word) of each, held pages, status
        each = 2 * 4 + (12 if case["tree"] else 0)
        return {"bytes": batch * (20 + nodes * each + 4 * ((nodes + page - 1) // page)), "flops": 0}
    if op == "write":
        width = case["kv"] * case["hd"]
        size = 2 if case["dtype"] == "bf16" else 4
        # in: keys, values, slots; out: codes and scales, and the cache's values, BF16
        new = case["tokens"] * (2 * width * size + 4 + 2 * width + 4 * width // _GROUP)
        kept = case["slots"] - case["tokens"]
        return {"bytes": new + max(kept, 0) * (2 * width + 4 * width // _GROUP) + case["slots"] * 2 * width * 2,
                "flops": 6 * case["tokens"] * 2 * width}
    if op == "attention":
        batch, nodes, hq, kv, hd = (case[n] for n in ("batch", "nodes", "hq", "kv", "hd"))
        # mean lengths and counts of the ragged batch (the first request is the longest)
        length = case["context"] * (1 + 0.5 * (batch - 1)) / batch
        count = nodes * (1 + 0.75 * (batch - 1)) / batch
        slot = 2 * kv * hd + 4 * kv * hd // _GROUP
        rows = batch * nodes * hq * hd * 2 * (3 if case["gate"] else 2)
        return {"bytes": batch * (length + count) * slot + rows,
                "flops": 4 * batch * count * hq * hd * (length + count)}
    batch, nodes, vocab = case["batch"], case["nodes"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    history = case["history"] * (1 + 0.5 * (batch - 1)) / batch
    bits = (vocab + 7) // 8 if case["mask"] else 0
    return {"bytes": batch * (nodes * (vocab * (size + 4) + bits) + 4 * history + 8 * 64),
            "flops": 6 * batch * nodes * vocab}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None  # whole numbers only
    if op == "write":
        out = []
        for name, x in (("k", s["key"]), ("v", s["value"])):
            x = x.double()
            codes = s["cache"][name][0].double().view(-1, x.shape[1], x.shape[2] // _GROUP, _GROUP)
            plane = s["cache"][name + "_scale"].double().t().reshape(codes.shape[:3])
            held = codes * plane[..., None]
            x = x.view(x.shape[0], *codes.shape[1:])
            scale = (x.abs().amax(-1, keepdim=True) / 127).to(torch.bfloat16).double()
            new = torch.round(x / torch.where(scale == 0, 1.0, scale)).clamp(-127, 127) * scale
            live = s["slots"] >= 0
            held[s["slots"][live].long()] = new[live]
            out.append(held.view(1, held.shape[0], *s["key"].shape[1:]))
        return out
    if op == "attention":
        q, page = s["q"].double(), s["page"]
        batch, nodes, hq, hd = q.shape
        kv = s["cache"]["k"].shape[2] // hd
        out = torch.zeros_like(q)
        lengths, counts = s["lengths"].tolist(), s["counts"].tolist()
        for b in range(batch):
            n, total = counts[b], lengths[b] + counts[b]
            if n == 0:
                continue
            times = [torch.arange(page, device=q.device) + int(p) * page for p in s["table"][b].tolist()]
            times = torch.cat(times)[:total]
            see = torch.ones((n, total), dtype=torch.bool, device=q.device)
            for i, word in enumerate(s["ancestors"][b, :n].tolist()):
                see[i, lengths[b]:] = torch.tensor([bool(word >> j & 1) for j in range(n)], device=q.device)
            for h in range(kv):
                kd, vd = (s["cache"][name][0, times, h * hd:(h + 1) * hd].double()
                          * s["cache"][name + "_scale"][h * hd // _GROUP:(h + 1) * hd // _GROUP, times].double()
                          .t().repeat_interleave(_GROUP, dim=1) for name in ("k", "v"))
                heads = slice(h * hq // kv, (h + 1) * hq // kv)
                scores = torch.einsum("nhd,td->nht", q[b, :n, heads], kd) / math.sqrt(hd)
                scores = scores.masked_fill(~see[:, None], -math.inf)
                out[b, :n, heads] = torch.einsum("nht,td->nhd", torch.softmax(scores, -1), vd)
        return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())
    x = s["logits"].double()
    batch, nodes, vocab = x.shape
    for b in range(batch):
        length, prompt = int(s["history_lengths"][b]), int(s["prompt_lengths"][b])
        before = torch.bincount(s["history"][b, :prompt].long(), minlength=vocab).double()
        said = torch.bincount(s["history"][b, prompt:length].long(), minlength=vocab).double()
        bias = torch.zeros(vocab, dtype=torch.float64, device=x.device)
        used = (s["bias_ids"][b] >= 0) & (s["bias_ids"][b] < vocab)
        bias[s["bias_ids"][b][used].long()] = s["bias"][b][used].double()
        for i in range(nodes):
            word = int(s["ancestors"][b, i])
            path = [j for j in range(nodes) if word >> j & 1]
            counts = said + torch.bincount(s["drafts"][b, path].long(), minlength=vocab)
            row, r = x[b, i], s["repetition"][b].double()
            row = torch.where(before + counts > 0, torch.where(row > 0, row / r, row * r), row)
            row = row - s["frequency"][b].double() * counts - s["presence"][b].double() * (counts > 0)
            row = (row + bias) / s["temperature"][b].double()
            if s["mask"] is not None:
                bits = s["mask"][b, i].view(torch.uint8)[:, None] >> torch.arange(8, device=x.device).to(torch.uint8)
                row = row.masked_fill((bits & 1).flatten()[:vocab] == 0, -math.inf)
            x[b, i] = row
    return x
