"""Logits processing on the GPU against the rules in 64 bits."""

import numpy as np
import pytest

from util import to_f32

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def oracle(x, r):
    """``(values, bound)``: the bound adds one FP32 rounding (2^-24 of the magnitude reached) per
    operation, of which a value passes at most seven."""
    batch, nodes, vocab = x.shape
    out, bound = np.empty(x.shape), np.empty(x.shape)
    for b in range(batch):
        length = 0 if r.get("history") is None else int(r["history_lengths"][b])
        prompt = int(r["prompt_lengths"][b]) if r.get("prompt_lengths") is not None else 0
        said, before = np.zeros(vocab), np.zeros(vocab)
        for i in range(length):
            v = int(r["history"][b, i])
            if 0 <= v < vocab:
                (before if i < prompt else said)[v] += 1
        bias = np.zeros(vocab)
        if r.get("bias_ids") is not None:
            for v, y in zip(r["bias_ids"][b], r["bias"][b]):
                if 0 <= v < vocab:
                    bias[v] = y
        rep, freq, pres, temp = (float(r[n][b]) if r.get(n) is not None else one
                                 for n, one in (("repetition", 1), ("frequency", 0), ("presence", 0), ("temperature", 1)))
        for i in range(nodes):
            count = said.copy()
            if r.get("drafts") is not None:
                for j in range(nodes):
                    v = int(r["drafts"][b, j])
                    if int(r["ancestors"][b, i]) >> j & 1 and 0 <= v < vocab:
                        count[v] += 1
            row = x[b, i]
            with np.errstate(invalid="ignore"):
                y = np.where((count > 0) | (before > 0), np.where(row > 0, row / rep, row * rep), row)
                size = np.abs(y) + abs(freq) * count + abs(pres) + np.abs(bias)
                y = (y - freq * count - pres * (count > 0) + bias) / temp
            if r.get("mask") is not None:
                bits = np.unpackbits(r["mask"][b, i].view(np.uint8), bitorder="little")[:vocab]
                y = np.where(bits == 1, y, -np.inf)
            out[b, i], bound[b, i] = y, 7 * EPS * size / temp
    return out, bound


def rules(rng, batch, nodes, vocab, room, names):
    few = lambda shape: rng.integers(0, max(vocab // 7, 2), shape)  # noqa: E731
    words = np.zeros((batch, nodes), np.uint64)
    for b in range(batch):
        for i in range(nodes):
            up = rng.integers(-1, i) if i else -1
            words[b, i] = np.uint64(1 << i) | (words[b, up] if up >= 0 else np.uint64(0))
    lengths = rng.integers(0, room + 1, batch)
    r = dict(history=few((batch, room)), history_lengths=lengths, prompt_lengths=lengths // 3,
             repetition=rng.uniform(0.8, 1.5, batch).astype(np.float32),
             frequency=rng.uniform(-0.5, 1, batch).astype(np.float32),
             presence=rng.uniform(-0.5, 1, batch).astype(np.float32),
             temperature=rng.uniform(0.2, 2, batch).astype(np.float32),
             bias_ids=rng.integers(-3, vocab + 3, (batch, 40)), bias=rng.normal(0, 5, (batch, 40)).astype(np.float32),
             drafts=few((batch, nodes)), ancestors=words,
             mask=rng.integers(-2 ** 31, 2 ** 31, (batch, nodes, (vocab + 31) // 32)).astype(np.int32))
    r["history"][:, ::5] = rng.integers(-9, vocab + 9, r["history"][:, ::5].shape)  # some outside the vocabulary
    r["mask"][-1, -1] = 0
    with_ = {"history": ("history", "history_lengths", "prompt_lengths"), "bias": ("bias_ids", "bias"),
             "drafts": ("drafts", "ancestors")}
    keep = [k for n in names for k in with_.get(n, (n,))]
    return {k: r[k] for k in keep}


ALL = ("history", "repetition", "frequency", "presence", "temperature", "bias", "drafts", "mask")


@pytest.mark.parametrize("batch,nodes,vocab,room,names", [
    (1, 1, 151936, 300, ALL), (2, 3, 5000, 64, ALL), (3, 64, 1237, 33, ALL), (5, 2, 4099, 1000, ALL),
    (1, 1, 1, 4, ALL), (2, 2, 31, 5, ALL), (4, 1, 4096, 0, ALL), (130, 5, 260, 50, ALL),
    (2, 2, 8192, 100, ("history", "repetition")), (2, 2, 515, 100, ("history", "frequency", "presence")),
    (2, 2, 512, 10, ("bias",)), (2, 2, 512, 10, ("mask",)), (2, 3, 512, 10, ("drafts", "presence")),
    (2, 2, 512, 10, ("temperature",)), (2, 2, 512, 10, ()),
])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_process_logits_rules(cuda_device, batch, nodes, vocab, room, names, dtype):
    import torch

    from qk_b200.sampling import process_logits

    rng = np.random.default_rng(vocab + nodes)
    r = rules(rng, batch, nodes, vocab, room, names)
    x = torch.from_numpy(rng.normal(0, 3, (batch, nodes, vocab)).astype(np.float32)).to(cuda_device)
    if vocab > 40:
        x[0, 0, 1:40:7] = 0.0
        x[0, 0, 2] = -float("inf")
    x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    given = {k: torch.from_numpy(v.view(np.int64) if v.dtype == np.uint64 else v).to(cuda_device) for k, v in r.items()}
    got = to_f32(process_logits(x, **given)).astype(np.float64)
    want, bound = oracle(to_f32(x).astype(np.float64), r)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    assert (np.abs(got[finite] - want[finite]) <= bound[finite]).all()
    if dtype == "f32":  # in place, and the same bits again
        again = process_logits(x, **given, out=x)
        assert again is x and np.array_equal(to_f32(x), got.astype(np.float32))


@pytest.mark.parametrize("vocab", [4089, 4095, 4097, 4104, 5003, 8185, 8191, 9001])
@pytest.mark.parametrize("nodes", [1, 9, 20])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_process_logits_ends_of_tiles(cuda_device, vocab, nodes, dtype, shift):
    """Rows that begin at every place of an access, vocabularies that end about a tile's end, logits that
    begin off an access, and a context with most of the vocabulary in it."""
    import torch

    from qk_b200.sampling import process_logits

    rng = np.random.default_rng(vocab + nodes)
    r = rules(rng, 2, nodes, vocab, 2 * vocab, ALL)
    r["history"] = rng.integers(0, vocab, (2, 2 * vocab))
    r["history_lengths"][0] = 2 * vocab
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    flat = torch.from_numpy(rng.normal(0, 3, 2 * nodes * vocab + 8).astype(np.float32)).to(cuda_device).to(dt)
    x = flat[shift:shift + 2 * nodes * vocab].view(2, nodes, vocab)
    given = {k: torch.from_numpy(v.view(np.int64) if v.dtype == np.uint64 else v).to(cuda_device) for k, v in r.items()}
    got = to_f32(process_logits(x, **given)).astype(np.float64)
    want, bound = oracle(to_f32(x).astype(np.float64), r)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    assert (np.abs(got[finite] - want[finite]) <= bound[finite]).all()


def test_process_logits_two_dimensions_and_repeated_biases(cuda_device):
    """[B, V] logits; of several biases of one token the last holds, however many there are."""
    import torch

    from qk_b200.sampling import process_logits

    x = torch.zeros((2, 100), device=cuda_device)
    ids = torch.full((2, 1024), 7)
    ids[1, 512:] = 8
    bias = torch.arange(2048, dtype=torch.float32).view(2, 1024)
    out = process_logits(x, bias_ids=ids, bias=bias)
    want = torch.zeros((2, 100))
    want[0, 7], want[1, 7], want[1, 8] = 1023, 1024 + 511, 2047
    assert torch.equal(out.cpu(), want)
    mask = torch.zeros((2, 4), dtype=torch.int32)
    assert torch.isneginf(process_logits(x, mask=mask)).all()
    assert process_logits(x[:0]).shape == (0, 100)


def test_process_logits_refusals(cuda_device):
    import torch

    from qk_b200.sampling import process_logits

    x = torch.zeros((2, 3, 64), device=cuda_device)
    with pytest.raises(TypeError):
        process_logits(x.half())
    for bad in (dict(history=torch.zeros((2, 4))), dict(bias_ids=torch.zeros((2, 4))), dict(drafts=torch.zeros((2, 3))),
                dict(mask=torch.zeros((2, 3, 3))), dict(repetition=torch.zeros(3)), dict(out=torch.zeros((2, 3, 64))),
                dict(bias_ids=torch.zeros((2, 1025)), bias=torch.zeros((2, 1025))),
                dict(history=torch.zeros((2, 1 << 20)), history_lengths=torch.zeros(2))):
        with pytest.raises(ValueError):
            process_logits(x, **bad)
    with pytest.raises(ValueError):
        process_logits(torch.zeros((2, 65, 8), device=cuda_device), drafts=torch.zeros((2, 65)),
                       ancestors=torch.zeros((2, 65)))
    with pytest.raises(ValueError):
        process_logits(x.cpu())
