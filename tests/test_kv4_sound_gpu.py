"""The cache held in 4 bits on the GPU: calls that the first tests of it did not make."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import plain_kv4 as P4
import plain_kv4_tight as tight
import test_kv4_gpu as first
from cuinfer_b200 import kernels
from test_kv4_gpu import BF16, F32, attend, case

pytestmark = pytest.mark.gpu


def check(c, out=None):
    """Against attention in 64 bits, within what the kernels' arithmetic may be off; rows behind the last request stay."""
    out = attend(c) if out is None else out
    kernels.check_error_flags(force=True)
    aligned = c["q"].data_ptr() % 16 == 0 and c["q"].stride(0) % 8 == 0
    want, allowed = tight.attention(c["q"], c["cache"], c["table"], c["starts"], c["lengths"], c["nq"], c["nkv"], c["d"], c["scale"], c["window"],
                                    rounded=c["q"].dtype == BF16, codes=aligned and c["d"] in (64, 128, 256))
    rows = c["starts"][-1]
    off = tight.worst(out, want, allowed, rows)
    print(f"{off:.3f} of what is allowed")
    assert off <= 1.0, f"{off:.2f} of what is allowed"
    assert (out[rows:] == 5.0).all(), "rows behind the last request are left as they are"


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens", [520, 1000])
@pytest.mark.parametrize("seed", [0, 1])
def test_pages_that_are_none_in_tiles_that_one_row_tile_no_longer_walks(monkeypatch, d, tokens, seed):
    """A CTA whose first row tile ends many key tiles before its second, with pages that are none in every tile: which ones is the second's
    business alone once the first has ended, and the first is still at its last tiles meanwhile."""
    monkeypatch.setattr(kernels, "kv4_prompt_shares", lambda *a: 1)
    rng = random.Random(seed)
    c = case([tokens + 24, 300], [tokens, 260], 2, 2, d, 16, BF16, seed=seed + d, spare_rows=1)
    c["table"] = [[-1 if rng.random() < 0.4 else p for p in row] for row in c["table"]]
    first = attend(c).clone()
    check(c, first)
    for _ in range(20):
        assert torch.equal(attend(c, torch.full_like(first, 5.0)), first)


# ---- the first tests' calls, within the bound of the kernels' arithmetic ------------------------------------------------------

@pytest.fixture
def within_the_bound(monkeypatch):
    monkeypatch.setattr(first, "check", check)


BOTH = pytest.mark.parametrize("dtype", [F32, BF16])
HEADS = pytest.mark.parametrize("heads", first.HEADS + [(4, 2, 192), (3, 1, 224), (4, 4, 256)])


@BOTH
@HEADS
def test_single_tokens(within_the_bound, dtype, heads):
    first.test_attention_of_single_tokens(dtype, heads, 48)


@BOTH
@HEADS
def test_prompts_and_mixed_steps(within_the_bound, dtype, heads):
    first.test_attention_of_prompts_and_mixed_steps(dtype, heads)


@BOTH
@pytest.mark.parametrize("window", [1, 33, 100])
@pytest.mark.parametrize("heads", [(4, 2, 128), (6, 2, 64), (2, 1, 96), (2, 1, 256)])
def test_windows(within_the_bound, dtype, window, heads):
    first.test_attention_in_a_window(dtype, window, heads)


@BOTH
@pytest.mark.parametrize("d", [64, 128, 96, 256])
def test_long_contexts(within_the_bound, dtype, d):
    first.test_attention_of_long_contexts(dtype, d)


@BOTH
@pytest.mark.parametrize("d", [64, 128, 96, 256])
@pytest.mark.parametrize("new", [1, 20])
def test_holes_and_empty_rows(within_the_bound, dtype, d, new):
    first.test_pages_that_are_none_rows_without_keys_and_empty_requests(dtype, d, new)


@pytest.mark.parametrize("heads", [(2, 1, 128), (12, 4, 64), (5, 1, 128)])
@pytest.mark.parametrize("shape", ["one long", "many", "portions", "bounds"])
def test_many_row_tiles(within_the_bound, heads, shape):
    first.test_prompts_of_many_row_tiles(heads, shape)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("shape", [(1, 0, 0), (8, 0, 0), (0, 5, 0), (0, 3, 8), (0, 592, 8)])
def test_shared_keys_of_single_tokens(within_the_bound, monkeypatch, d, window, shape):
    first.test_every_way_to_share_the_keys_of_single_tokens(monkeypatch, d, window, shape)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("shares", [2, 9])
def test_shared_keys_of_prompts(within_the_bound, monkeypatch, d, window, shares):
    first.test_prompts_whose_keys_are_shared(monkeypatch, d, window, shares)


@BOTH
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("cluster", [1, 8])
def test_without_tensor_cores(within_the_bound, monkeypatch, dtype, d, cluster):
    first.test_prompts_without_tensor_cores(monkeypatch, dtype, d, 0 if cluster == 1 else 60, cluster)


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("cluster", [1, 8])
def test_head_sizes_between(within_the_bound, monkeypatch, d, cluster):
    first.test_prompts_of_head_sizes_between(monkeypatch, d, 0 if cluster == 1 else 60, cluster)


@pytest.mark.parametrize("d", [96, 128])
@pytest.mark.parametrize("requests", [1, 3, 70])
def test_clusters_of_single_tokens(within_the_bound, d, requests):
    first.test_single_tokens_whose_keys_a_cluster_shares(d, requests)


def test_scales_that_are_not_positive(within_the_bound):
    first.test_a_scale_that_is_not_positive()


# ---- scores that differ by what the sums of the queries have in their lowest bits -----------------------------------------------

@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_scores_of_far_zero_points(d, new):
    """Two keys that are zero, one with codes and zero points of 15 and one of 0, under a query whose group's sum has 19 bits: both scores are
    exactly zero.  In units of a step every product is a multiple of 2^-10 and every sum below 2^12, so none of 24 bits is cut; the weights are equal,
    and the result is the values' mean, rounded once (2^-8) after weights of one."""
    groups = d // 32
    c = case([new + 1] * groups, [new] * groups, 1, 1, d, 16, BF16, seed=d)
    c["scale"] = 4.0
    q = torch.zeros_like(c["q"])
    for r in range(groups):
        q[c["starts"][r]:c["starts"][r + 1], 32 * r + 3], q[c["starts"][r]:c["starts"][r + 1], 32 * r + 14] = 258.0, 129 / 256
        q[c["starts"][r]:c["starts"][r + 1], 32 * r + 29] = 2.0 ** -10
    c["q"] = q
    raw = c["cache"].cpu().numpy()
    places = np.array(P4._places(d))[:, :, 0]
    for r in range(groups):
        block = raw[c["table"][r][0], 0, 0]
        for token in range(new + 1):
            code = 15 if token % 2 == 0 else 0
            for byte, shift, word in places[token]:
                block[byte] = block[byte] & ~(15 << shift) & 255 | code << shift
                block[word], block[word + 1] = 0x80 | code, 0x42             # a step of 64
    c["cache"] = torch.from_numpy(raw).to(first.DEV)
    out = attend(c).double().cpu()
    values = P4.unpack(c["cache"], d)[1]
    for r in range(groups):
        for i in range(new):
            want = values[c["table"][r][0], 0, :i + 2].mean(0)
            assert ((out[c["starts"][r] + i] - want).abs() <= 2.0 ** -8 * 1.01 * (want.abs() + (values[c["table"][r][0], 0, :i + 2].abs().mean(0) if new > 1 else 0))).all(), (r, i)
