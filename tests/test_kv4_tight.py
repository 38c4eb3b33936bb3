"""The bound that attention over the cache held in 4 bits is tested with, without a GPU: it lets the kernels' arithmetic through and nothing else."""
from __future__ import annotations

import pytest
import torch

import plain_kv4 as P4
import plain_kv4_tight as tight

HEADS = [32, 64, 96, 128, 160, 192, 224, 256]
NQ, NKV, LENGTHS = 6, 2, [130, 257, 300]


def make(d, new, rounded, seed=0, lengths=LENGTHS):
    g = torch.Generator().manual_seed(seed + d)
    pages = sum(-(-n // 16) for n in lengths) + 1
    cache = torch.randint(0, 256, (pages, NKV, 1, 18 * d), dtype=torch.uint8, generator=g)
    steps = torch.exp(0.3 * torch.randn(pages, NKV, 1, 2, d // 2, generator=g)) / 5
    words = ((steps.view(torch.int32) >> 16) & 0xFFF0) | torch.randint(5, 11, steps.shape, generator=g, dtype=torch.int32)
    both = torch.stack([(words & 255).to(torch.uint8), (words >> 8).to(torch.uint8)], -1).flatten(-2)
    cache[..., 8 * d:9 * d], cache[..., 17 * d:] = both[..., 0, :], both[..., 1, :]
    table, at = [], 1
    for n in lengths:
        table.append(list(range(at, at + -(-n // 16))))
        at += len(table[-1])
    starts = [0]
    for _ in lengths:
        starts.append(starts[-1] + new)
    q = torch.randn(starts[-1], NQ * d, generator=g) * 1.5
    return dict(q=q.bfloat16() if rounded else q, cache=cache, block_table=table, starts=starts, lengths=list(lengths), nq=NQ, nkv=NKV, d=d, scale=d ** -0.5)


def result(c, rounded, codes=False, **changes):
    return tight.attention(**{**c, **changes}, rounded=rounded, codes=codes)


@pytest.mark.parametrize("d", HEADS)
@pytest.mark.parametrize("rounded, codes", [(False, False), (True, False), (True, True)])
def test_wrong_results_are_rejected(d, rounded, codes):
    c = make(d, 1, rounded)
    want, allowed = result(c, rounded, codes)
    rows = want.shape[0]
    kind = torch.bfloat16 if rounded else torch.float32

    def off(wrong):
        return tight.worst(wrong.to(kind), want, allowed, rows)

    assert off(want) <= 0.5                                          # (one rounding)
    wrongs = {"zeros": torch.zeros_like(want), "a scale 1 % off": result(c, rounded, scale=c["scale"] * 1.01)[0]}
    for name, index in (("the last key left out", -1), ("the first page left out", 0)):
        table = [list(row) for row in c["block_table"]]
        lengths = list(c["lengths"])
        if index == 0:
            for row in table:
                row[0] = -1
            wrongs[name] = result(c, rounded, block_table=table)[0]
        else:                                                        # (positions do not enter the scores)
            wrongs[name] = result(c, rounded, lengths=[n - 1 for n in lengths])[0]
    keys = c["cache"].clone()
    keys[..., 0] ^= 1                                                # one code of a block off by one
    wrongs["heads exchanged"] = want.flip(1)
    if not rounded:
        wrongs["a result of bfloat16"] = want.bfloat16()
        wrongs["one code of a block off by one"] = result(c, rounded, cache=keys)[0]
    for name, wrong in wrongs.items():
        assert off(wrong) > 1.0, name


@pytest.mark.parametrize("d", [64, 96, 256])
@pytest.mark.parametrize("window", [0, 20])
def test_it_agrees_with_the_plain_form(d, window):
    """The two forms in 64 bits, with holes, rows in front of the first token and a request without rows."""
    c = make(d, 5, False, lengths=[40, 3, 33])
    c["block_table"][0][1] = -1
    c["block_table"][2] = c["block_table"][2][:2]
    want, _ = result(c, False, window=window)
    plain, _ = P4.attention(c["q"], c["cache"], c["block_table"], c["starts"], c["lengths"], NQ, NKV, d, c["scale"], window)
    assert torch.allclose(want, plain, rtol=1e-12, atol=1e-14)


def emulated(c, rounded):
    """The kernels' steps in torch: scores and sums in 32 bits, a weight (times the step) rounded to bfloat16 for the numerator."""
    step, code, zero = tight.planes(c["cache"], c["d"])
    numbers = (step * (code - zero)).float()
    out = torch.zeros(c["q"].shape[0], NQ, c["d"])
    for r, n in enumerate(c["lengths"]):
        index = torch.arange(n)
        at = torch.tensor(c["block_table"][r])[index // 16]
        for h in range(NQ):
            k, v = (numbers[at, h // (NQ // NKV), index % 16, :, i] for i in (0, 1))
            s = c["q"][r].float().reshape(NQ, -1)[h] @ k.T * c["scale"]
            p = torch.exp(s - s.max())
            w = p.bfloat16().float() if rounded else p
            out[r, h] = (w @ v) / p.sum()
    return out.bfloat16() if rounded else out


@pytest.mark.parametrize("d", HEADS)
@pytest.mark.parametrize("rounded", [False, True])
def test_the_arithmetic_of_the_kernels_is_let_through(d, rounded):
    c = make(d, 1, rounded, seed=7)
    want, allowed = result(c, rounded)
    assert tight.worst(emulated(c, rounded), want, allowed, want.shape[0]) <= 1.0
