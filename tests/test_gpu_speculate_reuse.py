"""A generation object that is used again starts anew."""

import numpy as np
import pytest

from test_gpu_speculate import VOCAB, model_of, prompts_of

pytestmark = pytest.mark.gpu


def test_prefill_starts_anew(cuda_device):
    """After a generation, and after one that ran out of pages, the same object gives a fresh one's tokens."""
    from qk_b200.paged import tree_attention
    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(6)
    first, second = prompts_of(rng, 3), [p[:9] for p in prompts_of(rng, 3)]

    def new():
        return SpeculativeGeneration(model, 3, 48, nodes=4, page_size=16, vocab=VOCAB, pages=6)

    fresh = new()
    fresh.prefill(second)
    want = fresh.generate(4)
    used = new()
    used.prefill([p[:9] for p in first])
    used.generate(5)
    used.prefill(second)
    assert used.generate(4) == want
    with pytest.raises(RuntimeError):
        used.generate(30)  # six pages do not hold three contexts
    with pytest.raises(ValueError):
        tree_attention.check_status()
    used.prefill(second)
    assert used.generate(4) == want


def test_padding_and_drafts_outside_the_vocabulary(cuda_device):
    """What nodes past the counts hold has no say, whatever it is; a draft outside the vocabulary is never kept."""
    import torch

    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(7)
    prompts = prompts_of(rng, 2)

    def drafts(history, lengths, nodes):
        tokens = torch.full((2, nodes), -1, dtype=torch.int32, device=cuda_device)
        tokens[:, :1] = torch.gather(history, 1, lengths[:, None].long() - 1)
        tokens[:, 1] = VOCAB + 7  # a draft, but no token
        tokens[1, 3] = 2 ** 31 - 1
        parents = torch.full((2, nodes), 2 ** 31 - 1, dtype=torch.int32, device=cuda_device)
        parents[:, :2] = torch.tensor([-1, 0])
        return tokens, parents, torch.full((2,), 2, dtype=torch.int32, device=cuda_device)

    gen = SpeculativeGeneration(model, 2, 48, nodes=4, page_size=16, vocab=VOCAB, drafts=drafts)
    gen.prefill(prompts)
    out = gen.generate(3)
    assert [len(o) - len(p) for o, p in zip(out, prompts)] == [3, 3]
    assert all(0 <= t < VOCAB for o in out for t in o)
    for bad in ([[0, VOCAB], [1]], [[0], [-1, 2]]):
        with pytest.raises(ValueError):
            gen.prefill(bad)
