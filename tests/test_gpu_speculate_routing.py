"""Speculative decoding over a model that selects its experts: a tree's passes and one-token passes agree where they
route alike, and route apart only at near ties."""

import numpy as np
import pytest

from test_gpu_speculate import VOCAB, prompts_of
from util import to_f32

pytestmark = pytest.mark.gpu


class Recorder:
    """The library, with what each expert selection chose of which logits."""

    def __init__(self, lib):
        self._lib, self.of, self.seen = lib, None, []

    def __getattr__(self, name):
        fn = getattr(self._lib, name)
        if name != "qk_router_select_shared":
            return fn

        def select(*args):
            status = fn(*args)
            k = self.of.model.cfg.top_k
            self.seen.append((self.of.ids[:, :k].sort(-1).values.cpu().numpy(), to_f32(self.of.router)))
            return status

        return select


def test_tree_and_single_passes_route_alike_but_for_near_ties(cuda_device, monkeypatch):
    """Top 2 of 16 experts. The two passes' activations differ by BF16 roundings (5e-2 of the largest, as for the
    model that routes to all): so may the router's logits, and a choice that differs must lie within twice that.
    Nodes whose path was routed alike in every layer keep the bound on their hidden states."""
    import torch

    from qk_b200 import _lib, speculate
    from qk_b200.decoder import StackConfig, SyntheticDecoder
    from qk_b200.speculate import SpeculativeGeneration

    model = SyntheticDecoder(StackConfig(layers=2, experts=16, top_k=2, qtype="Q4_K", context=96), cuda_device, seed=5)
    recorder = Recorder(_lib.load())
    monkeypatch.setattr(speculate._lib, "load", lambda: recorder)
    rng = np.random.default_rng(1)
    prompts = [p[:1] for p in prompts_of(rng, 8)]  # one token: all routing that reaches a node is recorded
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 3]] * 8, dtype=torch.int32, device=cuda_device)
    tokens = torch.from_numpy(rng.integers(0, VOCAB, (8, 7)).astype(np.int32)).to(cuda_device)
    tokens[:, 0] = torch.tensor([p[-1] for p in prompts])
    tree = SpeculativeGeneration(model, 8, 64, nodes=7, page_size=16, vocab=VOCAB)
    tree.prefill(prompts)
    recorder.of, recorder.seen = tree, []
    all_nodes = torch.full((8,), 7, dtype=torch.int32, device=cuda_device)
    got = to_f32(tree.forward(tokens, all_nodes, parents)[0]).reshape(8, 7, -1).copy()
    chosen = [(ids.reshape(8, 7, -1), logits.reshape(8, 7, -1)) for ids, logits in recorder.seen]
    one, alike, ties = torch.ones(8, dtype=torch.int32, device=cuda_device), 0, 0
    for node in range(7):
        path, j = [], node
        while j >= 0:
            path.append(j)
            j = int(parents[0, j])
        single = SpeculativeGeneration(model, 8, 64, nodes=1, page_size=16, vocab=VOCAB)
        single.prefill(prompts)
        same = np.ones(8, bool)
        for j in reversed(path):
            recorder.of, recorder.seen = single, []
            want = to_f32(single.forward(tokens[:, j:j + 1].contiguous(), one)[0])
            single.cached = single.cached + one
            for (ids, logits), (tree_ids, _) in zip(recorder.seen, chosen):
                for b in range(8):
                    if same[b] and (ids[b] != tree_ids[b, j]).any():
                        same[b] = False  # a first difference: between experts of nearly equal logits
                        apart = np.setxor1d(ids[b], tree_ids[b, j])
                        assert np.ptp(logits[b, apart]) <= 2 * 5e-2 * np.abs(logits[b]).max()
                        ties += 1
        for b in np.nonzero(same)[0]:
            alike += 1
            assert np.abs(got[b, node] - want[b]).max() <= 5e-2 * np.abs(want[b]).max()
    assert alike >= 40, f"{alike} of 56 nodes routed alike, {ties} near ties"
