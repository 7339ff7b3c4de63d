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


def same_rows(a, b):
    import torch

    return torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("batch", [1, 3])
def test_a_verified_token_has_the_projections_of_a_decode_step(cuda_device, batch):
    """The first layer's projections of one token, of the same hidden rows: equal bits in a decode step, in a
    pass of one node and from the operators themselves."""
    import torch

    from qk_b200.fp8 import fp8_matmul, rms_norm_fp8
    from qk_b200.speculate import SpeculativeGeneration

    model = model_of(cuda_device, layers=1)
    L = model.layers[0]
    g = torch.Generator(device=cuda_device).manual_seed(9)
    L.attn_norm = (1 + 0.3 * torch.randn(model.cfg.hidden, device=cuda_device, generator=g)).to(torch.bfloat16)
    gen = SpeculativeGeneration(model, batch, 64, nodes=1, page_size=16, vocab=VOCAB)
    gen.prefill([[7 + b] for b in range(batch)])
    tokens = torch.tensor([[7 + b] for b in range(batch)], dtype=torch.int32, device=cuda_device)
    gen.forward(tokens, torch.ones(batch, dtype=torch.int32, device=cuda_device))
    x = gen.embedding.index_select(0, tokens[:, 0].long())
    want = fp8_matmul(rms_norm_fp8(x, L.attn_norm, model.cfg.eps)[0], L.w_qkv)
    state = model.state(batch)
    state.x.copy_(x)
    state.step()
    assert torch.equal(bits(state.qkv), bits(want))
    assert torch.equal(bits(gen.qkv), bits(want))


def test_later_layers_of_a_verify_pass_take_codes_of_the_unrounded_norm(cuda_device):
    """In a pass of 2 x 3 nodes: the last layer's q, gate, k and v are the product of the codes that the residual
    add and norm leave, from the layer's own input."""
    import torch

    from qk_b200 import speculate
    from qk_b200.fp8 import Fp8Rows, fp8_matmul, quantize_fp8
    from qk_b200.speculate import SpeculativeGeneration

    model = model_of(cuda_device)
    gen = SpeculativeGeneration(model, 2, 64, nodes=3, page_size=16, vocab=VOCAB)
    gen.prefill([[5, 6], [7]])
    tokens = torch.tensor([[6, 1, 2], [7, 3, 4]], dtype=torch.int32, device=cuda_device)
    seen, attention = [], speculate.tree_attention

    def spied(*args, **kwargs):
        seen.append(attention(*args, **kwargs))
        return seen[-1]

    speculate.tree_attention = spied
    try:
        gen.forward(tokens, torch.tensor([3, 3], dtype=torch.int32, device=cuda_device))
    finally:
        speculate.tree_attention = attention
    width = model.cfg.hidden
    rows = Fp8Rows(gen.fp8.codes[:, :width], gen.fp8.scales)
    L = model.layers[-1]
    assert torch.equal(bits(gen.qkv), bits(fp8_matmul(rows, L.w_qkv)))
    assert torch.equal(bits(gen.a), bits(fp8_matmul(seen[-1].reshape(6, -1), L.w_o)))
    # all but a BF16 norm's codes: quantising the rounded row would give others
    norm = rows.codes.float() * rows.scales.t().repeat_interleave(128, 1)[:, :width]
    assert not same_rows(rows, quantize_fp8(norm.to(torch.bfloat16)))


@pytest.mark.parametrize("nodes", [4, 7])
def test_tree_hidden_states_match_token_by_token(cuda_device, nodes):
    """As for BF16 projections: each node of a tree agrees with feeding its path a token at a time."""
    import torch

    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(1)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (4, 19, 27)]
    tree = SpeculativeGeneration(model, 3, 64, nodes=nodes, page_size=16, vocab=VOCAB)
    tree.prefill(prompts)
    up = [-1, 0, 0, 1, 1, 2, 3][:nodes]
    parents = torch.tensor([up] * 3, dtype=torch.int32, device=cuda_device)
    tokens = torch.from_numpy(rng.integers(0, VOCAB, (3, nodes)).astype(np.int32)).to(cuda_device)
    tokens[:, 0] = torch.tensor([p[-1] for p in prompts])
    counts = torch.tensor([nodes, nodes - 2, 1], dtype=torch.int32, device=cuda_device)
    got = to_f32(tree.forward(tokens, counts, parents)[0]).reshape(3, nodes, -1).copy()
    one = torch.ones(3, dtype=torch.int32, device=cuda_device)
    for node in range(nodes):
        path, j = [], node
        while j >= 0:
            path.append(j)
            j = up[j]
        single = SpeculativeGeneration(model, 3, 64, nodes=1, page_size=16, vocab=VOCAB)
        single.prefill(prompts)
        for j in reversed(path):
            want = to_f32(single.forward(tokens[:, j:j + 1].contiguous(), one)[0])
            single.cached = single.cached + one
        for b in range(3):
            if node < int(counts[b]):
                assert np.abs(got[b, node] - want[b]).max() <= 0.1 * np.abs(want[b]).max()


def test_generated_tokens_are_greedy_choices(cuda_device):
    """As for BF16 projections: each generated token, scored by passes of one token, is the best one up to the
    difference between the two passes."""
    import torch

    from qk_b200.speculate import SpeculativeGeneration

    model, rng = model_of(cuda_device), np.random.default_rng(2)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (3, 12, 25)]
    spec = SpeculativeGeneration(model, 3, 60, nodes=6, page_size=16, vocab=VOCAB)
    spec.prefill(prompts)
    out = spec.generate(6)
    assert all(o[:len(p)] == p and 6 <= len(o) - len(p) <= 36 for o, p in zip(out, prompts))
    single = SpeculativeGeneration(model, 3, 60, nodes=1, page_size=16, vocab=VOCAB)
    one = torch.ones(3, dtype=torch.int32, device=cuda_device)
    for t in range(max(len(o) for o in out) - 1):
        tokens = torch.tensor([[o[min(t, len(o) - 1)]] for o in out], dtype=torch.int32, device=cuda_device)
        hidden, _ = single.forward(tokens, one)
        single.cached = single.cached + one
        logits = to_f32(torch.matmul(hidden, single.embedding.t()))
        for b, o in enumerate(out):
            if len(prompts[b]) - 1 <= t < len(o) - 1:
                assert logits[b, o[t + 1]] >= logits[b].max() - 0.1 * np.abs(logits[b]).max()


def expire(device):
    """A bounded wait of 200 microseconds at most that nothing ends, reported as a product's is."""
    from qk_b200 import _lib

    _lib.call("qk_fp8_expire", 200, _lib.stream_handle(device))


def test_a_wait_that_gave_up_is_reported_once(cuda_device):
    import torch

    from qk_b200.fp8 import check_status

    check_status(cuda_device)
    expire(cuda_device)
    with pytest.raises(RuntimeError):
        check_status(cuda_device)
    check_status(cuda_device)  # the report is cleared
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        expire(cuda_device)
    check_status(cuda_device)
    graph.replay()
    with pytest.raises(RuntimeError):
        check_status()
    check_status()


def test_generation_hands_back_no_tokens_of_a_product_that_gave_up(cuda_device):
    from qk_b200.generate import StaticGeneration
    from qk_b200.speculate import SpeculativeGeneration

    model = model_of(cuda_device, layers=1)
    spec = SpeculativeGeneration(model, 1, 64, nodes=2, page_size=16, vocab=VOCAB)
    spec.prefill([[5, 6]])
    expire(cuda_device)
    with pytest.raises(RuntimeError):
        spec.generate(1)
    assert len(spec.generate(1)[0]) >= 4  # asked once
    gen = StaticGeneration(model, 1, 8, 4, vocab=VOCAB, seed=1)
    expire(cuda_device)
    with pytest.raises(RuntimeError):
        gen.prefill()
    gen.prefill()
    expire(cuda_device)
    with pytest.raises(RuntimeError):
        gen.decode(1)
    gen.decode(1)
    gen.close()


def test_bf16_generation_does_not_ask(cuda_device):
    """What FP8 products reported is not a BF16 model's."""
    from qk_b200.fp8 import check_status
    from qk_b200.generate import StaticGeneration
    from qk_b200.speculate import SpeculativeGeneration

    model = model_of(cuda_device, layers=1, dense="bf16")
    expire(cuda_device)
    spec = SpeculativeGeneration(model, 1, 64, nodes=2, page_size=16, vocab=VOCAB)
    spec.prefill([[5, 6]])
    spec.generate(1)
    gen = StaticGeneration(model, 1, 8, 4, vocab=VOCAB, seed=1)
    gen.prefill()
    gen.decode(1)
    gen.close()
    with pytest.raises(RuntimeError):
        check_status(cuda_device)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_product_over_its_scales_is_refused(cuda_device, m):
    """The scales of x are read while the output is written, as its codes are."""
    import torch

    from qk_b200.fp8 import Fp8Rows, fp8_matmul, pack_fp8, quantize_fp8

    g = torch.Generator(device=cuda_device).manual_seed(m)
    w = pack_fp8(torch.randn((16, 512), device=cuda_device, generator=g).to(torch.bfloat16))
    rows = quantize_fp8(torch.randn((m, 512), device=cuda_device, generator=g).to(torch.bfloat16))
    store = torch.zeros(m * 64, device=cuda_device)
    scales = store[m * 24:m * 28].view(4, m)
    scales.copy_(rows.scales)
    rows = Fp8Rows(rows.codes, scales)
    want = fp8_matmul(rows, w, output_dtype=torch.float32)
    for at in (m * 24, m * 28 - 1, m * 9):  # all of them, the last, the first m
        with pytest.raises(ValueError):
            fp8_matmul(rows, w, out=store[at:at + m * 16].view(m, 16))
    for at in (m * 28, m * 8):  # behind them, and up to them
        assert torch.equal(fp8_matmul(rows, w, out=store[at:at + m * 16].view(m, 16)), want)
