"""The tree attention at full size, with calls in flight behind one another, and at the edges of its number
formats, against 64 bits on the GPU."""

import numpy as np
import pytest

from test_gpu_paged import random_pool, random_words

pytestmark = pytest.mark.gpu


def dense(q, cache, table, lengths, counts, words, page, gate=None, scale=None):
    """``softmax(q . k * scale) v`` of every node in 64 bits: FP64 ``[B, N, hq, hd]``. A product with a weight of
    zero is zero whatever it is multiplied by."""
    import torch

    batch, nodes, hq, hd = q.shape
    rows, time, width = cache["k"].shape
    kv, groups = width // hd, width // 32
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    scale = hd ** -0.5 if scale is None else scale
    for b in range(batch):
        n, c = int(lengths[b]), int(counts[b])
        if c == 0:
            continue
        t = torch.arange(n + c, device=q.device)
        slots = table[b].to(q.device).long()[t // page] * page + t % page
        r, s = slots // time, slots % time
        see = torch.ones((c, n + c), dtype=torch.bool, device=q.device)
        word = words[b, :c].to(q.device).long()
        see[:, n:] = ((word[:, None] >> torch.arange(c, device=q.device)) & 1).bool()
        kd, vd = ((cache[m][r, s].view(n + c, groups, 32).double()
                   * cache[m + "_scale"].view(rows, groups, time)[r, :, s].double()[..., None]).view(n + c, kv, hd)
                  for m in ("k", "v"))
        for h in range(kv):
            heads = slice(h * hq // kv, (h + 1) * hq // kv)
            x = torch.einsum("nhd,td->nht", q[b, :c, heads].double(), kd[:, h]) * scale
            x = x.masked_fill(~see[:, None], -torch.inf)
            w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)  # a node that sees nothing
            out[b, :c, heads] = torch.einsum("nht,td->nhd", w, vd[:, h])
    return out if gate is None else out * torch.sigmoid(gate.double())


def request_batch(g, rng, batch, nodes, hq, kv, hd, page, lengths, counts, sharp=1.5, gate=True):
    """The tensors of a call: ``dict`` of the arguments of tree_attention and counts, ragged as given."""
    import torch

    width = max(1, int(-(-(max(lengths) + nodes) // page)))
    cache = random_pool(g, 1, batch * width * page, kv, hd)
    table = torch.randperm(batch * width, generator=g, device=g.device).to(torch.int32).view(batch, width)
    q = (torch.randn((batch, nodes, hq, hd), generator=g, device=g.device) * sharp).to(torch.bfloat16)
    z = torch.randn((batch, nodes, hq, hd), generator=g, device=g.device).to(torch.bfloat16) if gate else None
    i32 = dict(dtype=torch.int32, device=g.device)
    words = torch.from_numpy(random_words(rng, batch, nodes).view(np.int64)).to(g.device)
    return dict(q=q, cache=cache, table=table, lengths=torch.tensor(lengths, **i32), ancestors=words, page_size=page,
                counts=torch.tensor(counts, **i32), gate=z)


def exactly(call):
    return dense(call["q"], call["cache"], call["table"], call["lengths"], call["counts"], call["ancestors"],
                 call["page_size"], call["gate"])


def off(out, want):
    """Per (request, node, head): the 2-norm of the difference over that of the wanted row."""
    return ((out.double() - want).norm(dim=-1) / want.norm(dim=-1).clamp(min=1e-30)).max().item()


def where_differs(out, first):
    """The place of the first differences: request, node, head and the channels there."""
    bad = (out.view(-1, *out.shape[2:]) != first.view(-1, *out.shape[2:])).nonzero()
    return f"{len(bad)} values, rows (request and node, head, channel) {bad[:6].tolist()} .. {bad[-3:].tolist()}"


# A row's error is the rounding to BF16 (at most 1.7e-3 for a norm, see the test of eleven bits), that of the
# scores (keys rounded to 11 bits: a relative 2^-12 / sqrt(3) of products that add up to a score of standard
# deviation s is s * 1.4e-4, which moves weights by as much and rows that few tokens make by all of it) and of
# weights and values (2.8e-4 together): 2e-3 for s = 1.5, and at s = 9 three deviations of 1.3e-3 more.
@pytest.mark.parametrize("sharp,most,bound", [(1.5, 16384, 3e-3), (9.0, 3000, 8e-3)])
def test_wide_trees_in_flight_behind_one_another(cuda_device, sharp, most, bound):
    """16 trees of up to 64 nodes over ragged prefixes (one empty, one request without nodes): several row tiles
    per KV head, idle quarters of them, one-tile units next to units of hundreds. Two sets of inputs are right by
    themselves, and passes that alternate between them with no wait give the same bits every time. With sharp
    scores the running maxima of single rows grow in the middle of a unit."""
    import torch

    from qk_b200.paged import tree_attention

    calls, wants = [], []
    for seed in (1, 2):
        rng, g = np.random.default_rng(seed), torch.Generator(device=cuda_device).manual_seed(seed)
        lengths, counts = rng.integers(1, most + 1, 16).tolist(), rng.integers(32, 65, 16).tolist()
        lengths[0], counts[0], lengths[1], counts[2] = most, 64, 0, 0
        calls.append(request_batch(g, rng, 16, 64, 16, 2, 256, 64, lengths, counts, sharp))
        wants.append(exactly(calls[-1]))
    firsts = []
    for call, want in zip(calls, wants):
        firsts.append(tree_attention(**call))
        torch.cuda.synchronize()
        assert off(firsts[-1], want) <= bound
    for _ in range(4):
        outs = [tree_attention(**calls[i % 2]) for i in range(60)]
        torch.cuda.synchronize()
        for i, out in enumerate(outs):
            assert torch.equal(out, firsts[i % 2]), f"pass {i}: {where_differs(out, firsts[i % 2])}"
        del outs
    tree_attention.check_status()


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("hd", [64, 256])
def test_drafts_that_are_not_finite_in_many_short_units(cuda_device, hd, which):
    """Several requests of one tile per SM, one behind the other: a draft that is not finite makes the nodes that
    see it NaN, and changes no bit of the requests before and behind it."""
    import torch

    from qk_b200.paged import tree_attention

    batch, nodes, kv = 7 * torch.cuda.get_device_properties(cuda_device).multi_processor_count // 2, 3, 2
    rng, g = np.random.default_rng(hd), torch.Generator(device=cuda_device).manual_seed(hd)
    call = request_batch(g, rng, batch, nodes, 4, kv, hd, 16, rng.integers(0, 13, batch).tolist(), [nodes] * batch)
    call["ancestors"] = torch.tensor([[1, 3, 5]], device=cuda_device).expand(batch, 3).contiguous()  # node 2 beside 1
    good = tree_attention(**call)
    hit = torch.arange(2, batch, 3, device=cuda_device)
    at = call["lengths"][hit].long() + 1  # node 1's token
    slots = call["table"][hit, at // 16].long() * 16 + at % 16
    groups = hd // 32
    call["cache"][which].view(kv, groups, -1)[1, groups - 1, slots] = float("nan")
    want = good.clone()
    touched = slice(None) if which == "k_scale" else slice(hd - 32, hd)
    want[hit, 1, 2:, touched] = float("nan")  # node 1 of the second KV head's query heads
    for _ in range(20):
        out = tree_attention(**call)
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))


def group_error(out, want):
    """The largest relative 2-norm of the error over the 32-channel groups of all rows, besides what BF16 rounds off
    where its own numbers are subnormal: 2^-134 of each value."""
    a, b = (x.double().reshape(-1, 32) for x in (out, want))
    assert not a.isnan().any()
    return (((a - b).norm(dim=-1) - 32 ** 0.5 * 2.0 ** -134) / b.norm(dim=-1).clamp(min=1e-300)).max().item()


# A group of 32 channels: the rounding to BF16 is within 2^-9 of each value; values, weights and scores add 2^-12 /
# sqrt(3) each, with which the weighted sum's terms err independently: below a third of that for any such group.
GROUP_BOUND = 4e-3


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("power", [16, 40, 100])
@pytest.mark.parametrize("length", [0, 30, 300])
def test_a_large_draft_counts_for_the_nodes_that_see_it_alone(cuda_device, hd, power, length):
    """A sibling whose value has another finite size, next to its neighbours' tokens, changes no bit of the rows
    that do not see it; those that do agree with 64 bits."""
    import torch

    from qk_b200.paged import tree_attention

    rng, g = np.random.default_rng(hd), torch.Generator(device=cuda_device).manual_seed(hd + length)
    call = request_batch(g, rng, 2, 6, 4, 2, hd, 16, [length, 77], [6, 6])
    call["ancestors"] = torch.tensor([[1, 3, 5, 11, 21, 37]], device=cuda_device).expand(2, 6).contiguous()
    good = tree_attention(**call)
    at = length + 1  # node 1, seen by nodes 1 and 3
    slot = int(call["table"][0, at // 16]) * 16 + at % 16
    call["cache"]["v_scale"][:, slot] *= 2.0 ** power
    out = tree_attention(**call)
    for node in range(6):
        assert torch.equal(out[0, node], good[0, node]) == (node not in (1, 3))
    assert torch.equal(out[1], good[1])
    assert group_error(out[0, [1, 3]], exactly(call)[0, [1, 3]]) <= GROUP_BOUND


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("power", [12, 24, 60, -60])
@pytest.mark.parametrize("at", [3, 40, 200])
def test_a_prefix_token_of_another_size_and_no_weight(cuda_device, hd, power, at):
    """A value 2^12 to 2^60 times its neighbours (or they that much larger than it), which every node sees with a
    weight of about exp(-90): it neither takes the other values' bits nor adds anything."""
    import torch

    from qk_b200.paged import tree_attention

    rng, g = np.random.default_rng(1), torch.Generator(device=cuda_device).manual_seed(hd)
    call = request_batch(g, rng, 1, 2, 4, 2, hd, 64, [260], [2], gate=False)
    call["q"] = (call["q"].abs() + 1).clamp(max=3.0)
    slot = int(call["table"][0, at // 64]) * 64 + at % 64
    cache = call["cache"]
    cache["k"][0, slot] = -127
    cache["k_scale"][:, slot] = 90.0 / 127 / hd ** 0.5
    others = torch.arange(cache["v_scale"].shape[1], device=cuda_device) != slot
    cache["v_scale"][:, ~others if power > 0 else others] *= 2.0 ** abs(power)
    assert group_error(tree_attention(**call), exactly(call)) <= GROUP_BOUND


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["tiny", "huge", "groups", "growing", "falling", "mixed"])
def test_values_of_many_sizes(cuda_device, hd, kind):
    """All values of one size, each channel group of its own, sizes that change along the cache or from token to
    token: every group of channels keeps its bits."""
    import torch

    from qk_b200.paged import tree_attention

    rng, g = np.random.default_rng(2), torch.Generator(device=cuda_device).manual_seed(hd)
    call = request_batch(g, rng, 3, 3, 8, 2, hd, 32, [700, 0, 65], [3, 3, 2])
    plane = call["cache"]["v_scale"]
    groups, slots = plane.shape
    t = torch.empty(slots, device=cuda_device)  # a slot's token
    for b in range(3):
        t.view(-1, 32)[call["table"][b].long()] = torch.arange(call["table"].shape[1] * 32, device=cuda_device).view(-1, 32).float()
    size = {"tiny": torch.full((groups, slots), -100.0), "huge": torch.full((groups, slots), 100.0),
            "groups": (torch.arange(groups) * -14.0 + 30)[:, None].expand(groups, slots),
            "growing": (t / 8).floor().expand(groups, slots), "falling": -(t / 8).floor().expand(groups, slots),
            "mixed": torch.randint(-40, 40, (groups, slots), generator=g, device=cuda_device)}[kind]
    plane.copy_((plane.double() * 2.0 ** size.to(cuda_device).double()).to(torch.bfloat16))
    assert group_error(tree_attention(**call), exactly(call)) <= GROUP_BOUND


def test_rows_past_the_fast_range_in_long_split_requests(cuda_device):
    """What is computed again is found through the parts of a request that many ranges share, at scales of the
    scores below and at zero, with values that are all zero beside."""
    import torch

    from qk_b200.paged import tree_attention

    rng, g = np.random.default_rng(3), torch.Generator(device=cuda_device).manual_seed(3)
    call = request_batch(g, rng, 1, 4, 16, 2, 256, 64, [6000], [4])
    call["cache"]["v_scale"][2, 5 * 64 + 7] *= 2.0 ** 30
    call["cache"]["v_scale"][5] = 0
    for scale in (None, 0.0, -0.05):
        out = tree_attention(**call, scale=scale)
        want = dense(call["q"], call["cache"], call["table"], call["lengths"], call["counts"], call["ancestors"], 64,
                     call["gate"], scale)
        assert (out[:, :, :8, 5 * 32:6 * 32] == 0).all()
        assert group_error(out, want) <= GROUP_BOUND


def test_reports_outlive_their_workspace_and_come_out_of_graphs(cuda_device):
    """A bad page is reported after a larger call has taken a larger workspace, from another stream, and from every
    replay of a graph, one that was captured without a call before it included; a report is raised once."""
    import torch

    from qk_b200.paged import TreeAttention

    attend = TreeAttention()
    rng, g = np.random.default_rng(4), torch.Generator(device=cuda_device).manual_seed(4)
    call = request_batch(g, rng, 2, 2, 4, 2, 64, 16, [40, 30], [2, 2])
    large = request_batch(g, rng, 40, 16, 4, 2, 64, 16, [40] * 40, [16] * 40)
    bad = dict(call, table=call["table"].clone().fill_(1 << 20))
    attend.check_status()
    attend(**bad)
    attend(**large)
    with pytest.raises(ValueError):
        attend.check_status()
    attend.check_status()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(**bad)
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        attend.check_status()
    held = dict(call, table=call["table"].clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = TreeAttention()(**held)
    graph.replay()
    attend.check_status()
    assert torch.equal(out, attend(**call))
    held["table"].copy_(bad["table"])
    for _ in range(2):
        graph.replay()
        with pytest.raises(ValueError):
            attend.check_status()
    held["table"].copy_(call["table"])
    graph.replay()
    attend.check_status()
    assert torch.equal(out, attend(**call))


def test_graphs_replayed_beside_one_another(cuda_device):
    """Two graphs, captured one after the other on torch's one capture stream, and calls outside them run on three
    streams at once: none writes into another's parts."""
    import torch

    from qk_b200.paged import tree_attention

    calls = []
    for seed in (5, 6, 7):
        rng, g = np.random.default_rng(seed), torch.Generator(device=cuda_device).manual_seed(seed)
        calls.append(request_batch(g, rng, 3, 4, 16, 2, 256, 64, [5000, 400, 3000], [4, 3, 4]))
    wants = [tree_attention(**c) for c in calls]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, call in zip(graphs, calls):
        with torch.cuda.graph(graph):
            outs.append([tree_attention(**call) for _ in range(10)])
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            outside = [tree_attention(**calls[2]) for _ in range(10)]
        torch.cuda.synchronize()
        for got, want in zip([*outs, outside], wants):
            assert all(torch.equal(o, want) for o in got)


def test_views_that_begin_off_sixteen_bytes(cuda_device):
    """Contiguous tokens, queries and gates at an odd address are copied, not refused."""
    import torch

    from qk_b200.paged import empty_pool, tree_attention, write_slots

    g = torch.Generator(device=cuda_device).manual_seed(8)

    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        view = flat[1:].view(x.shape)
        assert view.is_contiguous() and view.data_ptr() % 16
        return view.copy_(x)

    for dtype in (torch.bfloat16, torch.float32):
        key, value = (torch.randn((7, 2, 64), device=cuda_device, generator=g).to(dtype) for _ in range(2))
        slots = torch.arange(7, device=cuda_device)
        one, two = (empty_pool(2, 16, kv_heads=2, head_dim=64, device=cuda_device) for _ in range(2))
        write_slots(one, key, value, slots)
        write_slots(two, shifted(key), shifted(value), slots)
        assert all(torch.equal(one[n], two[n]) for n in one)
    call = request_batch(g, np.random.default_rng(8), 2, 3, 4, 2, 64, 16, [20, 9], [3, 2])
    want = tree_attention(**call)
    assert torch.equal(tree_attention(**dict(call, q=shifted(call["q"]), gate=shifted(call["gate"]))), want)


def test_outputs_over_queries_or_gates(cuda_device):
    """The output may be the queries' or the gate's own memory, also where it is computed again."""
    import torch

    from qk_b200.paged import tree_attention

    call = request_batch(torch.Generator(device=cuda_device).manual_seed(9), np.random.default_rng(9), 2, 3, 4, 2, 64, 16,
                         [200, 9], [3, 2])
    slot = int(call["table"][0, 6]) * 16 + 2
    call["cache"]["v_scale"][:, slot] *= 2.0 ** 40
    want = tree_attention(**call)
    for name in ("q", "gate"):
        own = call[name].clone()
        out = tree_attention(**dict(call, **{name: own}), out=own)
        assert out is own and torch.equal(out, want)
