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


# ---- keys next to the border of two codes ---------------------------------------------------------------------------------------

def rows_whose_roundings_add_up(d, T, nkv, seed):
    """Keys with one large value whose squares' sum loses nearly half a unit in every addition of a lane's chain, the lanes' exchange and eps:
    what is computed in 32 bits is above the exact value by as much as it can be.  The rotation's cosines put the normed value within some
    units of 14.5 steps, the border of two codes."""
    g = torch.Generator().manual_seed(seed)
    lanes, nearly = d // 16, 0.99 * 2.0 ** -24
    rows = torch.zeros(T, nkv, d, dtype=torch.float64)
    t, h = torch.arange(T)[:, None], torch.arange(nkv)[None]
    at = torch.randint(0, lanes, (T, nkv), generator=g)                  # the large value: the first of a lane's eight of the first half
    # sums of squares that reach the large value's lane one exchange after the other
    share = torch.zeros(T, nkv, lanes, dtype=torch.float64)
    o, count = lanes // 2, 1
    while o:
        for other in range(count):                                       # lanes that the partner at distance o has gathered
            bits = sum(((other >> i) & 1) * (lanes >> (i + 1)) for i in range(4))
            share[t, h, at ^ o ^ bits] = nearly / count
        o, count = o // 2, count * 2
    rows[..., :] = (share / 16).sqrt().repeat_interleave(8, -1).repeat(1, 1, 2)
    big = 1 + 0.004 * torch.rand(T, nkv, generator=g, dtype=torch.float64)     # (a unit of its square stays the same)
    for e in range(8):
        rows[t, h, 8 * at + e] = nearly ** 0.5 if e else 0.0
        rows[t, h, d // 2 + 8 * at + e] = (nearly / 8) ** 0.5
    rows *= big[..., None]
    rows[t, h, 8 * at] = big
    return rows.float(), nearly / d


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("norm", [True, False])
def test_keys_next_to_the_border_of_two_codes(d, norm):
    """The codes of a long prompt are those of 64 bits and of a call of few tokens, also where the errors of 32 bits add up next to a border."""
    T, nq, nkv, page = 12000, 1, 2, 16
    keys, eps = rows_whose_roundings_add_up(d, T, nkv, d)
    g = torch.Generator().manual_seed(1)
    gain = (1 + 0.2 * torch.rand(d, generator=g)).to(first.DEV) if norm else None
    size = 14.5 / (d ** 0.5 * gain.double().cpu()[:d // 2]) if norm else 14.5 / 1.01 * torch.ones(d // 2, dtype=torch.float64)
    angle = torch.zeros(600, d // 2, 2, dtype=torch.float64)
    angle[..., 0] = size * 2.0 ** -4 * (1 + (torch.rand(600, d // 2, generator=g, dtype=torch.float64) * 24 - 4) * 2.0 ** -24)
    table = angle.float().to(first.DEV)
    if not norm:                                                         # a border for a product of two 24-bit numbers, and its partner's
        keys = keys * 0 + 2.0 ** -10
        keys[..., ::8] = 1.01 * (1 + (torch.rand(T, nkv, d // 8, generator=g) * 8 - 4) * 2.0 ** -23)
        table[..., 1] = table[..., 0] * 2.0 ** -3
    qkv = torch.cat([torch.zeros(T, nq * d), keys.flatten(1), torch.zeros(T, nkv * d)], 1)
    positions = torch.arange(T, dtype=torch.int32) % 600
    pages = T // page + 1
    cache, small = (torch.zeros(kernels.kv4_cache_shape(pages, nkv, page, d), dtype=torch.uint8, device=first.DEV) for _ in range(2))
    dev, where, slots = qkv.to(first.DEV), positions.to(first.DEV), first.ints(list(range(T)))
    q_out = torch.empty(T, nq * d, device=first.DEV)
    kernels.qk_norm_rope_kv4_write(dev, where, slots, gain, gain, eps if norm else 0.0, table, d, cache, nq, nkv, d, q_out=q_out)
    for i in range(0, T, 1000):
        kernels.qk_norm_rope_kv4_write(dev[i:i + 1000], where[i:i + 1000], slots[i:i + 1000], gain, gain, eps if norm else 0.0, table, d, small, nq, nkv, d,
                                       q_out=q_out[:1000])
    _, k, _ = first.plain_rows(qkv, positions, gain, gain, eps if norm else 0.0, table, d, nq, nkv, d)
    want = torch.from_numpy(P4.held(k.numpy().astype(np.float32)))
    index = torch.arange(T)
    got, few = (P4.unpack(x, d)[0][index // page, :, index % page] for x in (cache, small))
    assert torch.equal(few, want)
    assert torch.equal(got, want), f"{int((got != want).any(-1).sum())} keys differ"


# ---- sizes at the ends of what the documentation allows --------------------------------------------------------------------------

@BOTH
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 31 - 40])
def test_the_largest_windows_with_rows_in_front_of_the_first_token(dtype, d, window):
    """A window of all keys: the rows of a request that brings more tokens than it holds see what they see without one."""
    c = case([12, 90, 0], [40, 90, 5], 4, 2, d, 16, dtype, window=window, seed=d)
    check(c)


@BOTH
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [1e-50, 1e-46, 1e-41, 1e-38, 1e-30])
def test_scales_next_to_zero(dtype, d, new, scale):
    """A positive scale that is zero in 32 bits, or not a normal number: every key weighs the same, and masked ones nothing."""
    c = case([90, 70], [new, new], 4, 2, d, 16, dtype, seed=3, window=30)
    c["scale"] = scale
    check(c)


@BOTH
@pytest.mark.parametrize("heads", [(300, 1, 64), (130, 1, 128), (70, 1, 96), (9, 1, 256), (258, 2, 32)])
def test_many_query_heads_to_a_key_head(dtype, heads):
    """A token's heads fill more than a row tile."""
    nq, nkv, d = heads
    check(case([70, 33, 5, 128], [3, 1, 5, 1], nq, nkv, d, 16, dtype, seed=d, spare_rows=1))


@BOTH
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("lens", ["exact", "bounds"])
def test_a_hundred_requests_of_every_kind(dtype, d, lens):
    rng = random.Random(d)
    new = [rng.choice([0, 1, 1, 2, 17, 40]) for _ in range(101)]
    lengths = [n + rng.choice([0, 3, 60]) for n in new]
    c = case(lengths, new, 4, 2, d, 16, dtype, seed=d, spare_rows=2)
    check(c, attend(c, lens=None if lens == "exact" else [sum(new) + 128] + [1] * 100, longest=None if lens == "exact" else 3000))


@BOTH
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_no_number_is_its_own_rows_business(dtype, d, new, bad):
    c = case([60, 300], [new, new], 6, 2, d, 16, dtype, seed=d)
    clean = attend(c).clone().reshape(2, new, 6, d)
    q = c["q"].clone()
    q[0, 1 * d + 7] = bad                                                # request 0, its first row, head 1
    q[new, 4 * d] = bad                                                  # request 1, its first row, head 4
    c["q"] = q
    got = attend(c, torch.full_like(c["out"], 5.0)).reshape(2, new, 6, d)
    for r, head in ((0, 1), (1, 4)):
        assert torch.isnan(got[r, 0, head]).all()
        got[r, 0, head] = clean[r, 0, head]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_recorded_step_of_a_long_model_for_any_batch(d):
    """One graph with the bounds of a recorded step and the longest context of its model, replayed for batches with and without single tokens, with
    requests that bring nothing, and with rows that belong to none of them."""
    R, T = 9, 96
    batches = [[40, 30, 0, 1, 2, 20, 3, 0, 0], [1] * 9, [96, 0, 0, 0, 0, 0, 0, 0, 0], [2, 3, 4, 5, 6, 7, 8, 9, 10], [0] * 9, [1, 0, 60, 0, 0, 0, 0, 1, 0]]
    c = case([400] * R, [T // R] * R, 4, 2, d, 16, BF16, seed=d, spare_rows=T - R * (T // R))
    table, starts, lengths = first.ints(c["table"]), first.ints([0] * (R + 1)), first.ints([0] * R)

    def call():
        kernels.paged_attention_kv4(c["q"], c["out"], c["cache"], table, starts, lengths, [T + 128] + [1] * (R - 1), 4, 2, d, c["scale"], max_seq_len=40960)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = random.Random(d)
    for new in batches + batches[::-1]:
        c["new"], c["lengths"] = new, [n + rng.randrange(400 - n) if n else 0 for n in new]
        c["starts"] = [sum(new[:i]) for i in range(R + 1)]
        starts.copy_(first.ints(c["starts"]))
        lengths.copy_(first.ints(c["lengths"]))
        c["out"].fill_(5.0)
        graph.replay()
        check(c, c["out"])
