"""Speculative decoding over paged caches: a tree's hidden states agree with feeding each path
token by token, and generated tokens are the model's greedy choices whatever was drafted."""

import numpy as np
import pytest

from util import to_f32

pytestmark = pytest.mark.gpu

VOCAB = 600


def model_of(device):
    from qk_b200.decoder import StackConfig, SyntheticDecoder

    # every expert takes every token: with a selection, a near tie in the router may go one way in a pass
    # of one token and another in a pass of several, and no bound on rounding holds across it
    return SyntheticDecoder(StackConfig(layers=2, experts=4, top_k=4, qtype="Q4_K", context=96), device, seed=5)


def prompts_of(rng, batch):
    return [rng.integers(0, VOCAB, n).tolist() for n in rng.integers(2, 30, batch)]


def test_tree_hidden_states_match_token_by_token(cuda_device):
    import torch

    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(1)
    prompts = prompts_of(rng, 3)
    tree = SpeculativeGeneration(model, 3, 64, nodes=7, page_size=16, vocab=VOCAB)
    tree.prefill(prompts)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 3]] * 3, dtype=torch.int32, device=cuda_device)
    tokens = torch.from_numpy(rng.integers(0, VOCAB, (3, 7)).astype(np.int32)).to(cuda_device)
    tokens[:, 0] = torch.tensor([p[-1] for p in prompts])
    counts = torch.tensor([7, 5, 1], dtype=torch.int32, device=cuda_device)
    got = to_f32(tree.forward(tokens, counts, parents)[0]).reshape(3, 7, -1).copy()
    one = torch.ones(3, dtype=torch.int32, device=cuda_device)
    for node in range(7):
        path, j = [], node
        while j >= 0:
            path.append(j)
            j = int(parents[0, j])
        single = SpeculativeGeneration(model, 3, 64, nodes=1, page_size=16, vocab=VOCAB)
        single.prefill(prompts)
        for j in reversed(path):
            want = to_f32(single.forward(tokens[:, j:j + 1].contiguous(), one)[0])
            single.cached = single.cached + one
        for b in range(3):
            if node < int(counts[b]):
                # the bound of the prefill's comparison with single steps: BF16 activations of two layers
                assert np.abs(got[b, node] - want[b]).max() <= 5e-2 * np.abs(want[b]).max()


@pytest.mark.parametrize("drafts", ["lookup", "branches"])
def test_generated_tokens_are_greedy_choices(cuda_device, drafts):
    """Each generated token, scored by single steps over the same sequence, is the best one up to the
    difference between the two passes; with drafts that hold the greedy continuation among wrong
    branches, several are kept per step."""
    import torch

    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(2)
    batch, context = 4, 60
    prompts = prompts_of(rng, batch)
    plain = SpeculativeGeneration(model, batch, context, nodes=1, page_size=16, vocab=VOCAB)
    plain.prefill(prompts)
    known = plain.generate(12)

    def branches(history, lengths, nodes):
        # 0 -> {wrong 1, right 2}, 2 -> {wrong 3, right 4}, 4 -> right 5
        tokens = torch.zeros((batch, nodes), dtype=torch.int32)
        for b, n in enumerate(lengths.tolist()):
            right = (known[b] + [0] * 8)[n:n + 3]
            tokens[b, :6] = torch.tensor([int(history[b, n - 1]), VOCAB - 1 - right[0], right[0], VOCAB - 1 - right[1],
                                          right[1], right[2]])
        parents = torch.tensor([[-1, 0, 0, 2, 2, 4]] * batch, dtype=torch.int32)
        return (tokens.to(cuda_device), parents.to(cuda_device),
                torch.full((batch,), 6, dtype=torch.int32, device=cuda_device))

    more = {} if drafts == "lookup" else {"drafts": branches}
    spec = SpeculativeGeneration(model, batch, context, nodes=6, page_size=16, vocab=VOCAB, **more)
    spec.prefill(prompts)
    out = spec.generate(6)
    grown = [len(o) - len(p) for o, p in zip(out, prompts)]
    assert all(6 <= g <= 36 for g in grown) and all(o[:len(p)] == p for o, p in zip(out, prompts))
    if drafts == "branches":
        assert sum(grown) >= 2 * 6 * batch  # of up to 4 per step
    single = SpeculativeGeneration(model, batch, context, nodes=1, page_size=16, vocab=VOCAB)
    one = torch.ones(batch, dtype=torch.int32, device=cuda_device)
    for t in range(max(len(o) for o in out) - 1):
        tokens = torch.tensor([[o[min(t, len(o) - 1)]] for o in out], dtype=torch.int32, device=cuda_device)
        hidden, _ = single.forward(tokens, one)
        single.cached = single.cached + one
        logits = to_f32(torch.matmul(hidden, single.embedding.t()))
        for b, o in enumerate(out):
            if len(prompts[b]) - 1 <= t < len(o) - 1:
                assert logits[b, o[t + 1]] >= logits[b].max() - 5e-2 * np.abs(logits[b]).max()


def test_rules_context_end_and_a_pool_that_runs_out(cuda_device):
    import torch

    from qk_b200.paged import tree_attention
    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(3)
    prompts = [rng.integers(0, VOCAB, 10).tolist() for _ in range(2)]
    banned = torch.arange(VOCAB, dtype=torch.int32, device=cuda_device)[:500].repeat(2, 1)
    rules = dict(bias_ids=banned, bias=torch.full((2, 500), -1e4, device=cuda_device),
                 presence=torch.full((2,), 100.0, device=cuda_device))
    gen = SpeculativeGeneration(model, 2, 24, nodes=4, page_size=16, vocab=VOCAB, rules=rules)
    gen.prefill(prompts)
    out = gen.generate(30)
    for o, p in zip(out, prompts):
        assert len(o) == 25  # the context's 24 tokens in the cache and the choice after them
        new = o[len(p):]
        assert all(500 <= t < VOCAB for t in new) and len(set(new)) == len(new)  # biased away, never twice
    small = SpeculativeGeneration(model, 2, 24, nodes=4, page_size=16, vocab=VOCAB, pages=2)
    small.prefill(prompts)
    with pytest.raises(RuntimeError):
        small.generate(30)
    with pytest.raises(ValueError):  # what the attention reported of it, once
        tree_attention.check_status()
