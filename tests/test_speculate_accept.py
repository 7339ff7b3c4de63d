"""The acceptance rule and the look-up drafts of speculative decoding against plain loops (CPU)."""

import numpy as np
import pytest


def words_of(parents, counts):
    batch, nodes = parents.shape
    words = np.zeros((batch, nodes), np.int64)
    for b in range(batch):
        for i in range(counts[b]):
            path, j = 0, i
            while j >= 0:
                path |= 1 << j
                j = int(parents[b, j])
            words[b, i] = path if path < 1 << 63 else path - (1 << 64)
    return words


@pytest.mark.parametrize("nodes,chain", [(1, False), (5, False), (12, True), (40, False), (64, True), (64, False)])
def test_accept_keeps_the_longest_path_of_choices(nodes, chain):
    import torch

    from qk_b200.speculate import accept

    rng = np.random.default_rng(nodes)
    batch = 30
    parents = np.array([[i - 1 if chain or rng.random() < 0.4 else rng.integers(-1, i) if i else -1
                         for i in range(nodes)] for _ in range(batch)])
    parents[:, 0] = -1
    counts = rng.integers(0, nodes + 1, batch)
    tokens, choices = (rng.integers(0, 3, (batch, nodes)) for _ in range(2))
    words = words_of(parents, counts)
    best, path, ranks, kept = accept(torch.from_numpy(tokens), None if chain else torch.from_numpy(parents),
                                     torch.from_numpy(words), torch.from_numpy(counts), torch.from_numpy(choices))
    long = 0
    for b in range(batch):
        good, depth = [False] * nodes, [0] * nodes
        for i in range(counts[b]):
            up = parents[b, i]
            good[i] = i == 0 or (up >= 0 and good[up] and tokens[b, i] == choices[b, up])
            depth[i] = 1 if up < 0 else depth[up] + 1
        if not counts[b]:
            assert kept[b] == 0 and not path[b].any()
            continue
        want = max((i for i in range(counts[b]) if good[i]), key=lambda i: (depth[i], -i))
        chain_of, j = [], want
        while j >= 0:
            chain_of.append(j)
            j = parents[b, j]
        chain_of.reverse()
        assert best[b] == want and kept[b] == len(chain_of)
        assert path[b].nonzero().flatten().tolist() == chain_of
        assert ranks[b][path[b]].tolist() == list(range(len(chain_of)))
        long = max(long, len(chain_of))
    assert long > 1 or nodes == 1


def test_lookup_drafts_follow_the_newest_tokens_last_place():
    import torch

    from qk_b200.speculate import lookup_drafts

    rows = [[5, 7, 8, 5, 9, 2, 5], [1, 2, 3], [4], [6, 6, 6, 6]]
    history = torch.zeros((4, 12), dtype=torch.int32)
    for b, row in enumerate(rows):
        history[b, :len(row)] = torch.tensor(row)
    tokens, parents, counts = lookup_drafts(history, torch.tensor([len(r) for r in rows]), 4)
    assert parents is None and counts.tolist() == [3, 1, 1, 1]
    assert tokens[0, :3].tolist() == [5, 9, 2] and tokens[1:, 0].tolist() == [3, 4, 6]


def test_accept_takes_a_parent_that_is_no_earlier_node_as_none():
    """As the step plan does: nodes past the counts may name anything, a node that names itself or a later one
    hangs on nothing and is not kept."""
    import torch

    from qk_b200.speculate import accept

    parents = torch.tensor([[7, 0, 0, 99, -5], [-1, 0, 3, 3, 2 ** 31 - 1]])
    counts = torch.tensor([3, 4])
    tokens = torch.tensor([[4, 1, 2, 0, 0], [4, 1, 2, 3, 0]])
    choices = torch.tensor([[2, 0, 5, 0, 0], [1, 2, 3, 0, 0]])
    fixed = parents.clone()
    fixed[0, 0] = fixed[0, 3] = fixed[0, 4] = fixed[1, 2] = fixed[1, 3] = fixed[1, 4] = -1
    words = torch.from_numpy(words_of(fixed.numpy(), counts.numpy()))
    best, path, ranks, kept = accept(tokens, parents, words, counts, choices)
    assert best.tolist() == [2, 1] and kept.tolist() == [2, 2]
    assert path.tolist() == [[True, False, True, False, False], [True, True, False, False, False]]
