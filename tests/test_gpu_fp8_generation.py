"""Generation with FP8 projections: prefill, speculative steps and decode steps of one model compute the same
function, whatever layout the attention's output comes in, and what the products report reaches the caller.

Tolerances. Between passes of different numbers of rows only the order of FP32 sums differs, but a code of 4 bits
may go the other way for a last bit of its input: hidden states and logits are compared with twice the room that
the same comparisons of BF16 projections have, 0.1 of the largest value. Where the passes have equal rows, equal
kernels run, and bits are compared.
"""

import numpy as np
import pytest

from util import to_f32

pytestmark = pytest.mark.gpu

VOCAB = 600


def model_of(device, layers=2, dense="fp8"):
    from qk_b200.decoder import StackConfig, SyntheticDecoder

    # every expert takes every token, so that no near tie of the router decides
    return SyntheticDecoder(StackConfig(layers=layers, experts=4, top_k=4, qtype="Q4_K", context=96, dense=dense), device, seed=5)


def bits(t):
    import torch

    return t.view(torch.int16)


@pytest.mark.parametrize("dense", ["fp8", "bf16"])
@pytest.mark.parametrize("batch", [1, 3])
def test_prefill_takes_any_layout_of_the_attention_output(cuda_device, monkeypatch, batch, dense):
    """Attention may return its output with the heads or the tokens outside; the values decide."""
    import torch

    from qk_b200.generate import StaticGeneration

    model = model_of(cuda_device, dense=dense)
    attention = torch.nn.functional.scaled_dot_product_attention
    got = {}
    for order in ("heads outside", "tokens outside"):
        def laid(*args, **kwargs):
            o = attention(*args, **kwargs)
            return o.contiguous() if order == "heads outside" else o.transpose(1, 2).contiguous().transpose(1, 2)

        monkeypatch.setattr(torch.nn.functional, "scaled_dot_product_attention", laid)
        gen = StaticGeneration(model, batch, 24, 4, vocab=VOCAB, seed=1)
        gen.prefill()
        got[order] = gen.logits.clone()
        gen.close()
    assert torch.equal(bits(got["heads outside"]), bits(got["tokens outside"]))


def test_prefill_of_one_sequence_matches_steps(cuda_device, monkeypatch):
    import torch

    from qk_b200.generate import StaticGeneration

    attention = torch.nn.functional.scaled_dot_product_attention
    monkeypatch.setattr(torch.nn.functional, "scaled_dot_product_attention", lambda *a, **k: attention(*a, **k).contiguous())
    model, prompt = model_of(cuda_device), 40
    gen = StaticGeneration(model, 1, prompt, 4, vocab=VOCAB, seed=1)
    gen.prefill()
    ref = StaticGeneration(model, 1, prompt, 4, vocab=VOCAB, seed=1)
    for t in range(prompt):
        ref.state.x.copy_(ref.embedding.index_select(0, ref.prompt_ids[:, t]))
        ref.state.positions.fill_(t)
        ref.state.step()
    ref._choose(0)
    a, b = to_f32(gen.logits), to_f32(ref.logits)
    assert np.abs(a - b).max() < 0.1 * np.abs(b).max()
    gen.close()
    ref.close()
