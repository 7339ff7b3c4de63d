"""Paged Q8 cache and draft trees on the GPU: the step plan, the append by slot and the tree
attention against plain 64-bit implementations."""

import math

import numpy as np
import pytest

from util import to_f32

pytestmark = pytest.mark.gpu


# ---- step plan ------------------------------------------------------------------------------


def plan_oracle(table, held, ring, span, lengths, counts, parents, nodes, page):
    """One step in plain Python, in request order; table and ring are changed."""
    batch, width = table.shape
    pages = len(ring)
    head, free = int(span[0]), int(span[1])
    slots = np.full((batch, nodes), -1, np.int64)
    positions = np.zeros((batch, nodes), np.int64)
    words = np.zeros((batch, nodes), np.uint64)
    held_out, status = np.array(held), np.zeros(batch, np.int64)
    asked = taken = 0
    returned = []
    for b in range(batch):
        length, count = max(int(lengths[b]), 0), min(max(int(counts[b]), 0), nodes)
        bad = length != lengths[b] or count != counts[b]
        need = -(-(length + count) // page)
        have = int(held[b])
        if need > have:
            asked += need - have if need <= width else 0
            if need > width:
                status[b] = 2
            elif asked > free:
                status[b] = 1
            else:
                for p in range(have, need):
                    table[b, p] = ring[(head + asked - (need - have) + p - have) % pages]
                taken += need - have
                held_out[b] = need
        else:
            returned += list(table[b, need:have])
            held_out[b] = need
        if bad:
            status[b] += 4
        for i in range(count):
            t = length + i
            if t // page < held_out[b]:
                slots[b, i] = int(table[b, t // page]) * page + t % page
            depth = i
            if nodes <= 64:
                path, j = 0, i
                while j >= 0:
                    path |= 1 << j
                    up = j - 1 if parents is None else int(parents[b, j])
                    if not -1 <= up < j:
                        up, status[b] = -1, status[b] | 8
                    j = up
                words[b, i] = path
                depth = bin(path).count("1") - 1
            positions[b, i] = length + depth
    for j, p in enumerate(returned):
        ring[(head + free + j) % pages] = p
    return slots, positions, words, held_out, np.array([(head + taken) % pages, free - taken + len(returned)]), status


def run_plan(dev, table, held, ring, span, lengths, counts, parents, nodes, page):
    import torch

    from qk_b200.paged import plan_step

    t = {n: torch.from_numpy(np.asarray(v, np.int32).copy()).to(dev)
         for n, v in dict(table=table, held=held, ring=ring, span=span, lengths=lengths, counts=counts).items()}
    up = None if parents is None else torch.from_numpy(np.asarray(parents, np.int32)).to(dev)
    p = plan_step(t["table"], t["held"], t["ring"], t["span"], t["lengths"], t["counts"], nodes=nodes, page_size=page,
                  parents=up)
    words = None if p.ancestors is None else p.ancestors.cpu().numpy().view(np.uint64)
    return (p.slots.cpu().numpy(), p.positions.cpu().numpy(), words, p.held.cpu().numpy(), p.span.cpu().numpy(),
            p.status.cpu().numpy(), t["table"].cpu().numpy(), t["ring"].cpu().numpy())


def check_plan(dev, table, held, ring, span, lengths, counts, parents, nodes, page):
    got = run_plan(dev, table, held, ring, span, lengths, counts, parents, nodes, page)
    table, ring = np.array(table), np.array(ring)
    want = plan_oracle(table, held, ring, span, lengths, counts, parents, nodes, page)
    for name, g, w in zip(("slots", "positions", "ancestors", "held", "span", "status"), got, want):
        if g is not None:
            np.testing.assert_array_equal(g, w, err_msg=name)
    np.testing.assert_array_equal(got[6], table, err_msg="table")
    np.testing.assert_array_equal(got[7], ring, err_msg="ring")
    return want, table, ring


@pytest.mark.parametrize("batch,nodes,page,tree", [(1, 1, 16, False), (3, 5, 16, True), (64, 64, 16, True),
                                                   (300, 8, 32, True), (7, 1500, 64, False), (2, 64, 1024, False)])
def test_plan_over_many_steps(cuda_device, batch, nodes, page, tree):
    """Requests grow, shrink (rejected drafts), end and run out of pages; no page is ever owned twice."""
    rng = np.random.default_rng(batch * 1000 + nodes)
    width = -(-(6 * nodes + 40) // page)
    pages = max(2, batch * width // 4)
    table, held = np.full((batch, width), -1), np.zeros(batch, np.int64)
    ring, span = rng.permutation(pages), np.array([pages - 1, pages])
    lengths = np.zeros(batch, np.int64)
    short = 0
    for _ in range(6):
        counts = rng.integers(0, nodes + 1, batch)
        parents = None
        if tree:
            parents = np.array([[rng.integers(-1, i) if i else -1 for i in range(nodes)] for _ in range(batch)])
        want, table, ring = check_plan(cuda_device, table, held, ring, span, lengths, counts, parents, nodes, page)
        held, span = want[3], want[4]
        short += int((want[5] == 1).sum())
        owned = [int(p) for b in range(batch) for p in table[b, :held[b]]]
        free = [int(ring[(span[0] + j) % pages]) for j in range(span[1])]
        assert sorted(owned + free) == list(range(pages))
        accepted = np.minimum(rng.integers(0, nodes + 1, batch), np.where(want[5] == 0, counts, 0))
        lengths = np.where(rng.random(batch) < 0.1, 0, lengths + accepted)
    assert short > 0 or batch < 64


def test_plan_reports_bad_input_and_a_narrow_table(cuda_device):
    # of 5 requests: a negative length, too many nodes, a parent that comes later, a table too
    # narrow, a good one
    lengths, counts = np.array([-3, 5, 17, 40, 16]), np.array([2, 9, 4, 4, 4])
    parents = np.array([[-1, 0, 1, 2], [-1, 0, 0, 0], [-1, 3, -7, 2], [-1, 0, 1, 2], [-1, -1, 0, 2]])
    held = np.array([0, 0, 1, 2, 1])
    table = np.array([[-1, -1], [-1, -1], [4, -1], [5, 6], [7, -1]])
    ring = np.array([0, 1, 2, 3, 9, 9, 9, 9, 8, 9])
    want, _, _ = check_plan(cuda_device, table, held, ring, np.array([8, 6]), lengths, counts, parents, 4, 16)
    assert list(want[5]) == [4, 4, 8, 2, 0]


@pytest.mark.parametrize("nodes", [4, 100])
def test_plan_beside_requests_that_outgrow_their_tables(cuda_device, nodes):
    """They take no page, and those behind them take the pages that the ring gives up: each page stays with one
    owner, and none is lost."""
    rng = np.random.default_rng(nodes)
    batch, page, width = 40, 16, 9
    pages = batch * width
    table, held = np.full((batch, width), -1), np.zeros(batch, np.int64)
    ring, span = rng.permutation(pages), np.array([pages - 5, pages])
    lengths = rng.integers(0, width * page + 20, batch)
    full = 0
    for _ in range(4):
        counts = rng.integers(0, nodes + 1, batch)
        want, table, ring = check_plan(cuda_device, table, held, ring, span, lengths, counts, None, nodes, page)
        held, span = want[3], want[4]
        full += int((want[5] == 2).sum())
        owned = [int(p) for b in range(batch) for p in table[b, :held[b]]]
        free = [int(ring[(span[0] + j) % pages]) for j in range(span[1])]
        assert sorted(owned + free) == list(range(pages))
        lengths = np.where(want[5] == 0, lengths + counts, rng.integers(0, width * page + 20, batch))
    assert full > 8


def test_plan_refusals():
    import torch

    from qk_b200.paged import empty_tables, plan_step

    table, held, ring, span = empty_tables(2, 4, 8, "cpu")
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        plan_step(table, held, ring, span, z, z, nodes=1, page_size=16)
    table, held, ring, span = empty_tables(2, 4, 8)
    for page in (8, 48, 2048):
        with pytest.raises(ValueError):
            plan_step(table, held, ring, span, z, z, nodes=1, page_size=page)
    with pytest.raises(ValueError):
        plan_step(table, held, ring, span, z[:1], z, nodes=1, page_size=16)
    with pytest.raises(ValueError):
        plan_step(table, held, ring, span, z, z, nodes=65, page_size=16, parents=torch.zeros(2, 65))
    with pytest.raises(TypeError):
        plan_step(table.long(), held, ring, span, z, z, nodes=1, page_size=16)


# ---- append by slot --------------------------------------------------------------------------


@pytest.mark.parametrize("kv,hd,rows,time", [(2, 256, 1, 96), (3, 128, 2, 64), (1, 64, 1, 32), (2, 16, 1, 32), (1, 8, 1, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_write_slots_writes_the_appends_bytes(cuda_device, kv, hd, rows, time, dtype):
    """Each token's codes and scales equal those of the framework's append at the same place, and
    padding, slots outside the cache and all other slots stay untouched."""
    import torch

    from qk_b200.attention_cache import CacheConfig, empty_cache, quantize
    from qk_b200.paged import write_slots

    g = torch.Generator(device=cuda_device).manual_seed(kv * hd)
    c = CacheConfig(kv_heads=kv, head_dim=hd, query_heads=kv, max_context=time)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    tokens, group = 13, min(32, hd)
    # keys and values as slices of one projection's output: strided tokens
    wide = (torch.randn((tokens, 2 * kv * hd + 16), device=cuda_device, generator=g) * 3).to(dt)
    key = wide[:, 16:16 + kv * hd].view(tokens, kv, hd)
    value = wide[:, 16 + kv * hd:].view(tokens, kv, hd)
    key[0] = 0
    cache = empty_cache(rows, c, cuda_device)
    for n in cache:
        cache[n].random_(0, 50, generator=g)
    before = {n: t.clone() for n, t in cache.items()}
    slots = torch.randperm(rows * time, generator=g, device=cuda_device)[:tokens].to(torch.int32)
    slots[3], slots[5], slots[6] = -1, rows * time, -100
    write_slots(cache, key, value, slots)
    for name, x in (("k", key), ("v", value)):
        codes, scale = quantize(x.reshape(tokens, kv * hd).contiguous(), group)
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < rows * time:
                r, t = divmod(s, time)
                before[name][r, t] = codes[i]
                before[name + "_scale"].view(rows, -1, time)[r, :, t] = scale[i]
        assert torch.equal(cache[name], before[name])
        assert torch.equal(cache[name + "_scale"], before[name + "_scale"])


def test_write_slots_takes_shapes_and_copies_uneven_strides(cuda_device):
    import torch

    from qk_b200.paged import empty_pool, write_slots

    g = torch.Generator(device=cuda_device).manual_seed(4)
    k = torch.randn((3, 5, 64, 2), device=cuda_device, generator=g).transpose(2, 3)  # [3, 5, 2, 64], channels strided
    v = torch.randn((5, 3, 2, 64), device=cuda_device, generator=g).transpose(0, 1)  # batch and node swapped
    slots = torch.randperm(32, device=cuda_device, generator=g)[:15].view(3, 5)
    one, two = (empty_pool(2, 16, kv_heads=2, head_dim=64, device=cuda_device) for _ in range(2))
    write_slots(one, k, v, slots)
    write_slots(two, k.reshape(15, 2, 64).contiguous(), v.reshape(15, 2, 64).contiguous(), slots.reshape(15))
    for n in one:
        assert torch.equal(one[n], two[n])
    write_slots(one, k[:0], v[:0], slots[:0])  # nothing to write
    with pytest.raises(ValueError):
        write_slots(one, k, v, slots.reshape(15))
    with pytest.raises(ValueError):
        write_slots(one, k[..., :32], v[..., :32], slots)
    with pytest.raises(TypeError):
        write_slots(one, k.half(), v.half(), slots)
    with pytest.raises(ValueError):
        write_slots({n: t.cpu() for n, t in one.items()}, k, v, slots)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("power", [0, 40, -40, 117, -110, -130])
def test_write_slots_codes_of_every_quotient(cuda_device, dtype, power):
    """Every significand of the group's maximum against every significand and power of two of a value, halves
    of a code among them, in the framework's codec byte for byte; also where scales are subnormal."""
    import torch

    from qk_b200.attention_cache import quantize
    from qk_b200.paged import empty_pool, write_slots

    significands = torch.arange(128, 256, dtype=torch.float32) / 128
    others = (significands[None] * 2.0 ** -torch.arange(9, dtype=torch.float32)[:, None]).reshape(-1)  # 1152
    others = others[:1116].view(36, 31)
    top = 127 * significands * 2  # scale: the significand times 2, rounded
    x = torch.cat([top[:, None, None].expand(128, 36, 1), others[None].expand(128, 36, 31) * top[:, None, None] / 1.99],
                  dim=2)  # values below the maximum, some past its 127.5th part
    exact = others[None] * significands[:, None, None] * 128  # and products that are whole and half codes
    x = torch.stack([x, torch.cat([top[:, None, None].expand(128, 36, 1), exact], dim=2)])
    x = (x.reshape(-1, 32) * torch.where(torch.arange(2 * 128 * 36) % 2 == 0, 1.0, -1.0)[:, None] * 2.0 ** power)
    x = x.to(cuda_device).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    tokens = x.shape[0] // 2
    key, value = x.view(2, tokens, 1, 32)
    cache = empty_pool(tokens // 16, 16, kv_heads=1, head_dim=32, device=cuda_device)
    write_slots(cache, key, value, torch.arange(tokens, device=cuda_device))
    for name, y in (("k", key), ("v", value)):
        codes, scale = quantize(y.reshape(tokens, 32).contiguous(), 32)
        assert torch.equal(cache[name].view(tokens, 32), codes)
        assert torch.equal(cache[name + "_scale"].view(-1), scale.view(-1))


@pytest.mark.parametrize("batch,selected,time,kv,hd", [(3, 7, 19, 3, 8), (1, 1, 1, 1, 16), (2, 1000, 333, 5, 32), (5, 64, 70, 7, 96),
                                                       (2, 9, 11, 3, 24)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_reads_of_odd_shapes(cuda_device, batch, selected, time, kv, hd, dtype):
    import torch

    from qk_b200.attention_cache import CacheConfig, read_quantized

    g = torch.Generator(device=cuda_device).manual_seed(selected)
    group = min(32, hd)
    groups = kv * hd // group
    codes = torch.randint(-128, 128, (batch, time, kv * hd), generator=g, device=cuda_device).to(torch.int8)
    scale = torch.randn((batch * groups, time), generator=g, device=cuda_device).to(torch.bfloat16)
    idx = torch.randint(-time - 3, time + 3, (batch, selected), generator=g, device=cuda_device).to(torch.int32)
    c = CacheConfig(kv_heads=kv, head_dim=hd, query_heads=kv, max_context=time)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    cache = dict(k=codes, k_scale=scale, v=codes, v_scale=scale)
    got = read_quantized(cache, "k", idx, c, dt)
    at = torch.where(idx < 0, idx + time, idx).clamp(0, time - 1).long()
    rows = torch.arange(batch, device=cuda_device)[:, None]
    want = codes[rows, at].float().view(batch, selected, groups, group)
    want = want * scale.view(batch, groups, time).permute(0, 2, 1)[rows, at].float()[..., None]
    assert torch.equal(got.reshape(-1), want.reshape(-1).to(dt))


# ---- tree attention ----------------------------------------------------------------------------


def random_pool(g, rows, time, kv, hd):
    import torch

    from qk_b200.attention_cache import quantize

    x = torch.randn((2, rows * time, kv * hd), device=g.device, generator=g)
    cache = {}
    for name, values in zip(("k", "v"), x):
        codes, scale = quantize(values, 32)
        cache[name] = codes.view(rows, time, kv * hd)
        cache[name + "_scale"] = scale.view(rows, time, -1).transpose(1, 2).reshape(-1, time).contiguous()
    return cache


def attention_oracle(q, cache, table, lengths, counts, words, page, gate, scale):
    """``(out, bound)`` in 64 bits; ``bound`` is the largest error that rounding keys, values,
    weights and the output to BF16 (2^-9 each) can cause: a score moves by at most
    ``d = 2^-9 scale sum |q k|``, the weights by a factor within ``exp(+-2 max d)``, the sum of
    weighted values by ``2^-9`` for each of its two factors, and the result rounds once more. FP32
    sums and exponentials add at most 2^-12 to that (thousands of terms of 2^-24)."""
    import torch

    batch, nodes, hq, hd = q.shape
    kv = cache["k"].shape[2] // hd
    rows, time = cache["k"].shape[:2]
    out = np.zeros((batch, nodes, hq, hd))
    bound = np.zeros_like(out)
    qd = q.double().cpu().numpy()
    eps = 2.0 ** -9
    for b in range(batch):
        total = int(lengths[b]) + int(counts[b])
        t = np.arange(total)
        slots = np.asarray(table[b])[t // page].astype(np.int64) * page + t % page
        idx = torch.from_numpy(slots).to(q.device)
        r, s = idx // time, idx % time
        kd, vd = (cache[n][r, s].double().view(total, kv, hd // 32, 32)
                  * cache[n + "_scale"].view(rows, -1, time)[r, :, s].double().view(total, kv, hd // 32, 1)
                  for n in ("k", "v"))
        kd, vd = (x.reshape(total, kv, hd).cpu().numpy() for x in (kd, vd))
        for i in range(int(counts[b])):
            seen = np.concatenate([np.arange(lengths[b]), lengths[b] + np.array(
                [j for j in range(int(counts[b])) if int(words[b, i]) >> j & 1], np.int64)]).astype(np.int64)
            if not len(seen):
                continue
            for h in range(hq):
                k, v = kd[seen, h // (hq // kv)], vd[seen, h // (hq // kv)]
                x = k @ qd[b, i, h] * scale
                d = float(eps * scale * (np.abs(k) @ np.abs(qd[b, i, h])).max())
                w = np.exp(x - x.max())
                w /= w.sum()
                o, mass = w @ v, w @ np.abs(v)
                z = 1.0 if gate is None else 1 / (1 + np.exp(-gate[b, i, h].double().cpu().numpy()))
                out[b, i, h] = o * z
                bound[b, i, h] = z * (eps * np.abs(o) + (2 * eps + math.expm1(2 * d) + 2.0 ** -12) * mass) + 1e-6
    return out, bound


def random_words(rng, batch, nodes):
    words = np.zeros((batch, nodes), np.uint64)
    for b in range(batch):
        for i in range(nodes):
            up = rng.integers(-1, i) if i else -1
            words[b, i] = np.uint64(1 << i) | (words[b, up] if up >= 0 else np.uint64(0))
    return words


def check_attention(dev, seed, batch, nodes, hq, kv, hd, page, lengths, counts, words=None, gate=True, static=False,
                    poison=False, scale=None):
    import torch

    from qk_b200.paged import tree_attention

    rng = np.random.default_rng(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths, counts = np.asarray(lengths), np.asarray(counts)
    width = max(1, int(-(-(lengths.max() + nodes) // page)))
    rows = batch if static else 1
    spare = 0 if static else 2
    cache = random_pool(g, rows, (batch * width // rows + spare) * page, kv, hd)
    if static:
        table = np.arange(batch * width).reshape(batch, width)
        table = np.stack([rng.permutation(row) for row in table])
    else:
        table = rng.permutation(batch * width + spare)[:batch * width].reshape(batch, width)
    words = random_words(rng, batch, nodes) if words is None else words
    if poison:  # whatever no node may see: other pages, slots past the drafts, and table entries past them
        time = cache["k"].shape[1]
        used = np.zeros(rows * time, bool)
        for b in range(batch):
            t = np.arange(lengths[b] + counts[b])
            used[table[b][t // page] * page + t % page] = True
            table[b, -(-(lengths[b] + counts[b]) // page):] = 2 ** 30
        free = torch.from_numpy(~used).to(dev).view(rows, 1, time)
        for n, bad in (("k_scale", float("nan")), ("v_scale", float("inf"))):
            cache[n].view(rows, -1, time).masked_fill_(free, bad)
    q = (torch.randn((batch, nodes, hq, hd), device=dev, generator=g) * 1.5).to(torch.bfloat16)
    z = torch.randn((batch, nodes, hq, hd), device=dev, generator=g).to(torch.bfloat16) if gate else None
    out = tree_attention(q, cache, torch.from_numpy(table.astype(np.int32)).to(dev), torch.from_numpy(lengths),
                         torch.from_numpy(words.view(np.int64)), page_size=page, counts=torch.from_numpy(counts), gate=z,
                         scale=scale)
    tree_attention.check_status()
    want, bound = attention_oracle(q, cache, table, lengths, counts, words, page, z, hd ** -0.5 if scale is None else scale)
    got = to_f32(out).astype(np.float64)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    # typical rather than worst case: the roundings are independent, each uniform within 2^-9, and
    # a score of standard deviation 1.5 moves by 1.5 * 2^-9 / sqrt(3): 2.7e-3 in all, twice that
    if np.abs(want).max() > 0:
        assert np.linalg.norm(got - want) <= 5.4e-3 * np.linalg.norm(want)
    for b in range(batch):
        assert (got[b, counts[b]:] == 0).all()
    return got


@pytest.mark.parametrize("hq,kv,hd", [(16, 2, 256), (24, 2, 256), (6, 2, 128), (8, 8, 128), (5, 1, 64), (4, 4, 64)])
@pytest.mark.parametrize("nodes,page", [(1, 256), (7, 16), (64, 64)])
def test_tree_attention_heads_nodes_and_pages(cuda_device, hq, kv, hd, nodes, page):
    lengths = [130, 1, 63, 64, 65, 300]
    counts = [nodes, nodes, max(nodes // 2, 1), nodes, 1, nodes]
    check_attention(cuda_device, hq * hd + nodes, 6, nodes, hq, kv, hd, page, lengths, counts)


@pytest.mark.parametrize("gate,static,page", [(True, False, 16), (False, False, 32), (False, True, 64), (True, True, 16)])
def test_tree_attention_sees_only_what_it_may(cuda_device, gate, static, page):
    """Empty requests, counts of zero, words with no bit, NaN and infinite scales and table entries
    out of range wherever a node may not look."""
    rng = np.random.default_rng(5)
    words = random_words(rng, 6, 9)
    words[4] = 0               # no prefix and nothing of the tree: zero
    words[5, 3:] = 0           # the prefix alone
    got = check_attention(cuda_device, 11, 6, 9, 16, 2, 256, page, [0, 100, 37, 0, 0, 70], [9, 0, 4, 0, 9, 9], words,
                          gate=gate, static=static, poison=True)
    assert (got[4] == 0).all() and np.abs(got[0]).max() > 0


def test_tree_attention_long_prefix_split_over_the_gpu(cuda_device):
    check_attention(cuda_device, 21, 1, 16, 16, 2, 256, 256, [20011], [16])
    check_attention(cuda_device, 22, 2, 1, 16, 2, 256, 64, [9000, 17], [1, 1], gate=False)


def test_tree_attention_batch_with_few_tokens(cuda_device):
    rng = np.random.default_rng(9)
    check_attention(cuda_device, 23, 70, 3, 8, 4, 128, 16, rng.integers(0, 90, 70), rng.integers(0, 4, 70))


def test_tree_attention_steep_and_flat_scores(cuda_device):
    """A scale of zero averages the values; scores that grow along the cache move the running
    maximum again and again."""
    import torch

    from qk_b200.paged import tree_attention

    check_attention(cuda_device, 24, 2, 5, 16, 2, 256, 64, [500, 77], [5, 5], scale=0.0)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    cache = random_pool(g, 1, 1024, 2, 256)
    grow = torch.linspace(0.01, 40.0, 1024, device=cuda_device)
    cache["k"].fill_(100)
    cache["k_scale"].copy_((grow / 100).to(torch.bfloat16).expand(16, 1024))
    q = torch.full((1, 2, 16, 256), 1 / 16, dtype=torch.bfloat16, device=cuda_device)
    q[0, 1] = -q[0, 1]
    table = torch.arange(4, dtype=torch.int32, device=cuda_device)[None]
    words = torch.tensor([[1, 2]], device=cuda_device)
    out = to_f32(tree_attention(q, cache, table, torch.tensor([1020]), words, page_size=256))
    lengths, counts = np.array([1020]), np.array([2])
    want, bound = attention_oracle(q, cache, table.cpu().numpy(), lengths, counts, words.cpu().numpy().view(np.uint64), 256,
                                   None, 1 / 16)
    assert (np.abs(out - want) <= bound).all()


@pytest.mark.parametrize("hq,kv,hd", [(8, 1, 256), (6, 2, 128), (3, 3, 64)])
def test_tree_attention_rounds_operands_to_eleven_bits(cuda_device, hq, kv, hd):
    """The output's own rounding to BF16 (uniform within 2^-9, 1.1e-3 on average, for mantissas spread
    over [1, 2) at most 1.7e-3 in all) and little else: keys, values and weights carry 11 bits, so each
    adds an eighth of what BF16 operands would, under 1e-3 together."""
    import torch

    from qk_b200.paged import tree_attention

    g = torch.Generator(device=cuda_device).manual_seed(hd)
    cache = random_pool(g, 1, 2048, kv, hd)
    q = (torch.randn((1, 4, hq, hd), device=cuda_device, generator=g) * 1.5).to(torch.bfloat16)
    table = torch.arange(8, dtype=torch.int32, device=cuda_device)[None]
    words = torch.tensor([[1, 3, 5, 15]])
    out = to_f32(tree_attention(q, cache, table, torch.tensor([2000]), words, page_size=256)).astype(np.float64)
    want, _ = attention_oracle(q, cache, table.cpu().numpy(), np.array([2000]), np.array([4]),
                               words.numpy().view(np.uint64), 256, None, hd ** -0.5)
    assert np.linalg.norm(out - want) <= 2.0e-3 * np.linalg.norm(want)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -100, 1e-30, 1e-6, 3e4, 1e20, 2.0 ** 100])
def test_tree_attention_values_of_any_size(cuda_device, hd, size):
    """Values far outside FP16's range, also next to tiles of ordinary ones, scale the output alone."""
    import torch

    from qk_b200.paged import tree_attention

    g = torch.Generator(device=cuda_device).manual_seed(7)
    cache = random_pool(g, 1, 256, 2, hd)
    q = torch.randn((1, 1, 4, hd), device=cuda_device, generator=g).to(torch.bfloat16)
    table = torch.arange(4, dtype=torch.int32, device=cuda_device)[None]
    scale = torch.full((256,), size, device=cuda_device)
    scale[64:128] = 1.0  # a tile of ordinary values
    cache["v_scale"].copy_((cache["v_scale"].float() * scale).to(torch.bfloat16))
    args = (table, torch.tensor([255]), torch.tensor([[1]]))
    out = to_f32(tree_attention(q, cache, *args, page_size=64)).astype(np.float64)
    want, bound = attention_oracle(q, cache, table.cpu().numpy(), np.array([255]), np.array([1]),
                                   np.array([[1]], np.uint64), 64, None, hd ** -0.5)
    assert np.isfinite(out).all()
    slack = bound - 1e-6 + 2.0 ** -120  # the absolute part of the bound is for values near one
    assert (np.abs(out - want) <= slack).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 2.0 ** 125])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_tree_attention_drafts_that_are_not_finite(cuda_device, hd, bad, which):
    """A draft whose key or value is not finite makes the nodes that see it NaN (in its group of
    channels for a value), and changes no bit of the others."""
    import torch

    from qk_b200.paged import tree_attention

    g = torch.Generator(device=cuda_device).manual_seed(6)
    cache = random_pool(g, 1, 512, 2, hd)
    q = torch.randn((1, 6, 4, hd), device=cuda_device, generator=g).to(torch.bfloat16)
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device=cuda_device)
    words = torch.tensor([[1, 3, 5, 11, 21, 37]])  # nodes 1 and 3 see node 1
    args = (table, torch.tensor([300]), words)
    good = tree_attention(q, cache, *args, page_size=128)
    groups = hd // 32
    slot = int(table[0, 301 // 128]) * 128 + 301 % 128
    plane = cache[which].view(2, groups, 512)
    plane[1, groups - 1, slot] = bad  # KV head 1, the last group of its channels
    out = tree_attention(q, cache, *args, page_size=128)
    for node in range(6):
        for head in range(4):
            row, was = out[0, node, head], good[0, node, head]
            if node in (1, 3) and head >= 2:
                nan = torch.isnan(row)
                assert nan[-32:].all() and (which == "k_scale" or torch.equal(row[:-32], was[:-32]))
                assert which == "v_scale" or nan.all()
            else:
                assert torch.equal(row, was)


def test_tree_attention_strided_queries_and_streams(cuda_device):
    """Queries as a slice of the projection's output, and calls on two streams at once: each has a
    workspace of its own."""
    import torch

    from qk_b200.paged import tree_attention

    g = torch.Generator(device=cuda_device).manual_seed(8)
    cache = random_pool(g, 1, 64 * 128, 2, 256)
    wide = torch.randn((2, 6, 16 * 256 + 64), device=cuda_device, generator=g).to(torch.bfloat16)
    q = wide[..., 64:].view(2, 6, 16, 256)
    table = torch.randperm(128, device=cuda_device, generator=g).to(torch.int32).view(2, 64)
    words = (2 << torch.arange(6, device=cuda_device)).sub(1).expand(2, 6)
    lengths = torch.tensor([4000, 3333], device=cuda_device)
    first = tree_attention(q, cache, table, lengths, words, page_size=64)
    dense = tree_attention(q.contiguous(), cache, table, lengths, words, page_size=64)
    assert torch.equal(first, dense)
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(tree_attention(q, cache, table, lengths, words, page_size=64))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_tree_attention_captured_before_a_larger_call(cuda_device):
    """A graph keeps the workspace that it was captured with, also when a later call needs a larger one."""
    import torch

    from qk_b200.paged import TreeAttention

    attention = TreeAttention()
    g = torch.Generator(device=cuda_device).manual_seed(9)
    cache = random_pool(g, 1, 64 * 32, 2, 128)
    table = torch.randperm(32, device=cuda_device, generator=g).to(torch.int32).view(2, 16)
    lengths = torch.tensor([900, 77], device=cuda_device, dtype=torch.int32)
    words = (2 << torch.arange(48, device=cuda_device)).sub(1).expand(2, 48).contiguous()
    q = torch.randn((2, 48, 8, 128), device=cuda_device, generator=g).to(torch.bfloat16)
    call = lambda n: attention(q[:, :n], cache, table, lengths, words[:, :n].contiguous(), page_size=64)  # noqa: E731
    small = call(2)
    stream, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
    few, one = q[:, :2].contiguous(), words[:, :2].contiguous()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        attention(few, cache, table, lengths, one, page_size=64)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = attention(few, cache, table, lengths, one, page_size=64)
        call(48)
        junk = torch.full((1 << 26,), 255, dtype=torch.uint8, device=cuda_device)  # takes what was given back
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, small) and junk[0] == 255


def test_tree_attention_offsets_past_32_bits(cuda_device):
    """Codes more than 4 GiB into the pool."""
    import torch

    from qk_b200.paged import empty_pool, tree_attention, write_slots

    pages = 4 * 1024 * 1024 // 1024 + 300
    cache = empty_pool(pages, 1024, kv_heads=8, head_dim=128, device=cuda_device)
    small = empty_pool(2, 1024, kv_heads=8, head_dim=128, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    k, v = torch.randn((2, 1, 1500, 8, 128), device=cuda_device, generator=g)
    at = torch.arange(1500, device=cuda_device)
    last = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32, device=cuda_device)
    q = torch.randn((1, 3, 16, 128), device=cuda_device, generator=g).to(torch.bfloat16)
    outs = []
    for pool, table in ((cache, last), (small, torch.tensor([[1, 0]], dtype=torch.int32, device=cuda_device))):
        write_slots(pool, k, v, (table[0, at // 1024] * 1024 + at % 1024)[None])
        outs.append(tree_attention(q, pool, table, torch.tensor([1497]), torch.tensor([[1, 3, 7]]), page_size=1024))
    assert torch.equal(outs[0], outs[1]) and outs[0].abs().max() > 0


def test_tree_attention_reports_a_page_outside_the_cache(cuda_device):
    import torch

    from qk_b200.paged import TreeAttention, empty_pool

    attend = TreeAttention()
    cache = empty_pool(4, 16, kv_heads=1, head_dim=64, device=cuda_device)
    q = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16, device=cuda_device)
    attend(q, cache, torch.tensor([[0, 9]]), torch.tensor([20]), torch.tensor([[1]]), page_size=16)
    with pytest.raises(ValueError):
        attend.check_status()
    attend.check_status()  # reported once


def test_tree_attention_refusals(cuda_device):
    import torch

    from qk_b200.paged import empty_pool, tree_attention

    cache = empty_pool(4, 16, kv_heads=2, head_dim=64, device=cuda_device)
    table, one = torch.zeros((1, 4), dtype=torch.int32), torch.ones((1, 2), dtype=torch.int64)

    def call(q=torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16, device=cuda_device), table=table, lengths=torch.tensor([3]),
             words=one, page=16, cache=cache, **more):
        return tree_attention(q, cache, table, lengths, words, page_size=page, **more)

    call()
    with pytest.raises(TypeError):
        call(q=torch.zeros((1, 2, 4, 64), device=cuda_device))
    for bad in (dict(q=torch.zeros((1, 65, 4, 64), dtype=torch.bfloat16, device=cuda_device), words=torch.ones((1, 65))),
                dict(q=torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device=cuda_device)),
                dict(q=torch.zeros((1, 2, 4, 96), dtype=torch.bfloat16, device=cuda_device)),
                dict(table=table[0]), dict(lengths=torch.tensor([3, 3])), dict(words=one[:, :1]), dict(page=24),
                dict(page=8), dict(page=128), dict(cache={n: t.cpu() for n, t in cache.items()}),
                dict(gate=torch.zeros((1, 2, 4, 32), device=cuda_device))):
        with pytest.raises(ValueError):
            call(**bad)
