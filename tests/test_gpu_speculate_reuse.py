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
