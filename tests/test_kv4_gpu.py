"""The cache held in 4 bits on the GPU: appending, reading back, attention, and the engine over it."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import plain_kv4 as P4
import plain_qwen3 as P
import traces
from conftest import TOLERANCE, random_tokens
from cuinfer_b200 import kernels

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- appending and reading back ------------------------------------------------------------------------------------------

def plain_rows(qkv, positions, q_gain, k_gain, eps, table, rotary, nq, nkv, d):
    """queries, keys, values float64 [T, heads, d] after norm and rotation; the keys rounded once to 32 bits."""
    x = qkv.double().cpu()[:, :(nq + 2 * nkv) * d].reshape(qkv.shape[0], nq + 2 * nkv, d)
    q, k, v = x[:, :nq].clone(), x[:, nq:nq + nkv].clone(), x[:, nq + nkv:]
    out = []
    for rows, gain in ((q, q_gain), (k, k_gain)):
        if gain is not None:
            rows = rows / torch.sqrt((rows ** 2).mean(-1, keepdim=True) + float(np.float32(eps))) * gain.double().cpu()
        if rotary:
            half = rotary // 2
            at = positions.cpu().long().clamp(0, table.shape[0] - 1)
            c, s = table.double().cpu()[at][:, None].unbind(-1)
            a, b = rows[..., :half].clone(), rows[..., half:rotary].clone()
            rows = torch.cat((a * c - b * s, b * c + a * s, rows[..., rotary:]), -1)
        out.append(rows)
    return out[0], out[1].float().double(), v


def rope_table(positions, rotary, theta=10000.0):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(DEV)


WRITES = [  # T, nq, nkv, d, page, rotary, norm
    (1, 1, 1, 32, 16, 32, True), (3, 4, 2, 64, 16, 64, True), (17, 16, 8, 128, 16, 128, True), (40, 5, 1, 96, 48, 96, False),
    (300, 4, 2, 128, 32, 128, True), (257, 6, 3, 64, 16, 64, False), (9, 2, 2, 256, 16, 64, True), (300, 8, 4, 64, 64, 0, True),
    (33, 3, 1, 160, 32, 20, True), (2049, 2, 1, 128, 16, 128, True), (513, 7, 3, 128, 16, 0, False),
    # enough heads for several to a warp
    (1300, 4, 2, 128, 16, 128, True), (1201, 6, 3, 64, 16, 64, True), (1700, 2, 2, 256, 32, 256, True), (1300, 4, 2, 128, 16, 0, True),
    (1300, 4, 2, 128, 16, 64, True), (1600, 5, 1, 128, 16, 128, False), (1600, 1, 3, 64, 48, 0, False)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", WRITES)
@pytest.mark.parametrize("order", ["page by page", "anywhere"])
def test_write_and_read(dtype, sizes, order):
    T, nq, nkv, d, page, rotary, norm = sizes
    rng = random.Random(T * d + nq)
    pages = (2 * T + page - 1) // page + 2
    if order == "anywhere":
        slots = rng.sample(range(pages * page), T)
        for i in rng.sample(range(T), T // 7):
            slots[i] = -1
    else:
        ids = rng.sample(range(pages), pages)
        first = rng.randrange(page)
        slots = [ids[(first + i) // page] * page + (first + i) % page for i in range(T)]
    width = (nq + 2 * nkv) * d
    qkv = rand(T, width + 32, seed=T + d, dtype=dtype) * torch.exp(0.5 * rand(width + 32, seed=5)).to(dtype)
    positions = torch.tensor([rng.randrange(0, 700) for _ in range(T)], dtype=torch.int32)
    q_gain, k_gain = ((1 + rand(d, seed=s, scale=0.3)).to(dtype).to(DEV) if norm else None for s in (1, 2))
    table = rope_table(600, rotary) if rotary else None              # (positions beyond it read its last row)
    cache = torch.randint(0, 256, kernels.kv4_cache_shape(pages, nkv, page, d), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).to(DEV)
    before = cache.cpu()
    dev = qkv.to(DEV)[:, :width]                                     # rows of a wider tensor
    q_out = torch.full((T, nq * d), 7.0, dtype=dtype, device=DEV)
    args = (positions.to(DEV), ints(slots), q_gain, k_gain, 1e-5, table, rotary, cache, nq, nkv, d)
    kernels.qk_norm_rope_kv4_write(dev, *args, q_out=q_out)
    assert torch.equal(dev.cpu(), qkv[:, :width])                    # nothing of the rows is changed ...
    q, k, v = plain_rows(qkv, positions, q_gain, k_gain, 1e-5, table, rotary, nq, nkv, d)
    # a query is a product of the norm's factor (d / 32 + 8 additions in 32 bits, a reciprocal root good to 2^-21), a gain and a
    # rotation of two products: under 2^-17 of the pair's size; then it is rounded once
    near = q.abs()
    if rotary:
        half = rotary // 2
        pair = near[..., :half] + near[..., half:rotary]
        near = torch.cat((pair, pair, near[..., rotary:]), -1) * 1.5
    allowed = near * 2.0 ** -17 + (2.0 ** -8 * 1.01 * q.abs() if dtype == BF16 else 0.0)
    assert ((q_out.double().cpu().reshape(T, nq, d) - q).abs() <= allowed + 1e-30).all()
    # the cache: exactly the plain format
    got = cache.cpu()
    want = before.clone().numpy()
    places = np.array(P4._places(d))
    for t, slot in enumerate(slots):
        if slot < 0 or T > 300 and t % 37:
            continue
        p, b, token = slot // page, slot % page // 16, slot % 16
        for h in range(nkv):
            keys, values = P4.read_block(got[p, h, b].numpy(), d)
            for rows, held, plane in ((k, keys, 0), (v, values, 1)):
                for g in range(d // 32):
                    x = rows[t, h, 32 * g:32 * g + 32].numpy().astype(np.float32)
                    codes, word = P4.quantise_group(x)
                    assert [P4.value(c, word) for c in codes] == held[token, 32 * g:32 * g + 32].tolist(), (t, h, plane, g)
    # what belongs to no slot of the call is untouched
    mask = np.zeros(want.shape, dtype=np.uint8)
    for slot in slots:
        if slot >= 0:
            m = mask[slot // page, :, slot % page // 16]
            for plane in (0, 1):
                byte, shift, word = (places[slot % 16, :, plane, i] for i in range(3))
                for b, s in zip(byte, shift):
                    m[:, b] |= np.uint8(15 << s)
                m[:, word], m[:, word + 1] = 255, 255
    assert not ((got.numpy() ^ want) & ~mask).any()
    # ... every value of it
    at = torch.tensor([s if s >= 0 else 0 for s in slots])
    for rows, hold in zip((k, v), P4.unpack(cache, d)):
        there = hold[at // page, :, at % page]
        expect = torch.from_numpy(P4.held(rows.numpy().astype(np.float32)))
        live = torch.tensor(slots) >= 0
        assert torch.equal(there[live], expect[live])
    # reading back, in either type; a slot that is none leaves its row
    for kind in (F32, BF16):
        keys, values = (torch.full((T, nkv * d), -3.0, dtype=kind, device=DEV) for _ in range(2))
        kernels.kv4_read(cache, ints(slots), keys, values, nkv, d)
        for got_rows, hold in zip((keys, values), P4.unpack(cache, d)):
            rows = got_rows.double().cpu().reshape(T, nkv, d)
            assert torch.equal(rows[live], hold[at // page, :, at % page][live]) and (rows[~live] == -3).all()
    # in place: the queries of the rows are replaced, keys and values stay
    kernels.qk_norm_rope_kv4_write(dev, *args)
    assert torch.equal(dev[:, :nq * d], q_out) and torch.equal(dev[:, nq * d:].cpu(), qkv[:, nq * d:width]) and torch.equal(cache.cpu(), got)


def test_write_of_groups_that_do_not_fit_and_of_zeros():
    nq, nkv, d = 2, 2, 64
    qkv = rand(20, (nq + 2 * nkv) * d, seed=3)
    qkv[0, nq * d + 5] = float("nan")
    qkv[1, (nq + nkv) * d + 40] = float("inf")
    qkv[2, (nq + nkv) * d + 70] = -float("inf")
    qkv[3, nq * d:] = 0.0
    qkv[4, nq * d:] = 2.0 ** 127
    qkv[5, nq * d:] = 1.999 * 2.0 ** 126 * torch.sign(qkv[5, nq * d:])
    qkv[6, nq * d:] *= 2.0 ** -130
    cache = torch.zeros(kernels.kv4_cache_shape(3, nkv, 16, d), dtype=torch.uint8, device=DEV)
    dev = qkv.to(DEV)
    kernels.qk_norm_rope_kv4_write(dev, ints([0] * 20), ints(range(9, 29)), None, None, 0.0, None, 0, cache, nq, nkv, d)
    keys, values = torch.empty(20, nkv * d, device=DEV), torch.empty(20, nkv * d, device=DEV)
    kernels.kv4_read(cache, ints(range(9, 29)), keys, values, nkv, d)
    for rows, first in ((keys, nq * d), (values, (nq + nkv) * d)):
        x = qkv[:, first:first + nkv * d].reshape(20, nkv, d // 32, 32).numpy()
        got = rows.cpu().reshape(20, nkv, d // 32, 32).numpy()
        for index in np.ndindex(20, nkv, d // 32):
            codes, word = P4.quantise_group(x[index])
            np.testing.assert_array_equal(np.array([P4.value(c, word) for c in codes], dtype=np.float32), got[index])


def test_write_and_read_of_nothing_and_of_slots_outside():
    cache = torch.full(kernels.kv4_cache_shape(2, 1, 16, 32), 9, dtype=torch.uint8, device=DEV)
    empty = torch.empty(0, 96, device=DEV)
    kernels.qk_norm_rope_kv4_write(empty, ints([]), ints([]), None, None, 0.0, None, 0, cache, 1, 1, 32)
    kernels.kv4_read(cache, ints([]), torch.empty(0, 32, device=DEV), torch.empty(0, 32, device=DEV), 1, 32)
    rows = rand(3, 96, seed=1).to(DEV)
    kernels.qk_norm_rope_kv4_write(rows, ints([0] * 3), ints([-1, 32, 2 ** 31 - 1]), None, None, 0.0, None, 0, cache, 1, 1, 32)
    assert (cache == 9).all()
    keys, values = torch.ones(3, 32, device=DEV), torch.ones(3, 32, device=DEV)
    kernels.kv4_read(cache, ints([-5, 32, 2 ** 31 - 1]), keys, values, 1, 32)
    assert (keys == 1).all() and (values == 1).all()


# ---- attention ---------------------------------------------------------------------------------------------------------

def make_cache(pages, nkv, page, d, seed, scale=1.0):
    """Random codes with steps of about ``scale`` / 5: the numbers that random keys and values are held as."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.randint(0, 256, kernels.kv4_cache_shape(pages, nkv, page, d), dtype=torch.uint8, generator=g)
    steps = torch.exp(0.3 * torch.randn(*cache.shape[:3], 2, d // 2, generator=g)) * scale / 5
    words = (((steps.view(torch.int32) >> 16) & 0xFFF0) | torch.randint(5, 11, steps.shape, generator=g, dtype=torch.int32))
    low, high = (words & 255).to(torch.uint8), (words >> 8).to(torch.uint8)
    both = torch.stack([low, high], -1).flatten(-2)
    cache[..., 8 * d:9 * d], cache[..., 17 * d:] = both[..., 0, :], both[..., 1, :]
    return cache.to(DEV)


def case(lengths, new, nq, nkv, d, page, dtype, window=0, seed=0, spare_rows=0, sharp=1.5, holes=()):
    rng = random.Random(seed)
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3
    ids = rng.sample(range(pages), pages)
    stride = max(need + [1]) + 1
    table, at = [], 0
    for count in need:
        table.append(ids[at:at + count] + [-1] * (stride - count))
        at += count
    for r, i, page_id in holes:
        table[r][i] = page_id
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = rand(starts[-1] + spare_rows, nq * d + 64, seed=seed + 1, scale=sharp, dtype=dtype).to(DEV)[:, :nq * d]
    cache = make_cache(pages, nkv, page, d, seed)
    out = torch.full((starts[-1] + spare_rows, nq * d), 5.0, dtype=dtype, device=DEV)
    return dict(q=q, out=out, cache=cache, table=table, starts=starts, lengths=lengths, new=new, nq=nq, nkv=nkv, d=d, window=window, scale=d ** -0.5)


def attend(c, out=None, longest=None, lens=None, table=None):
    out = c["out"] if out is None else out
    kernels.paged_attention_kv4(c["q"], out, c["cache"], ints(c["table"]) if table is None else table, ints(c["starts"]), ints(c["lengths"]),
                                lens or c["new"], c["nq"], c["nkv"], c["d"], c["scale"], c["window"], max_seq_len=longest or max(c["lengths"] + [1]))
    return out


def check(c, out=None):
    out = attend(c) if out is None else out
    kernels.check_error_flags(force=True)
    want, allowed = P4.attention(c["q"], c["cache"], c["table"], c["starts"], c["lengths"], c["nq"], c["nkv"], c["d"], c["scale"], c["window"],
                                 rounded=c["q"].dtype == BF16)
    rows = c["starts"][-1]
    got = out.double().cpu().reshape(want.shape)
    off = ((got - want).abs() / allowed.clamp(min=1e-12))[:rows]
    assert not torch.isnan(off).any() and float(off.max()) <= 1.0, f"{float(off.max()):.2f} of what is allowed"
    assert (got[rows:] == 5.0).all(), "rows behind the last request are left as they are"


HEADS = [(2, 1, 128), (8, 2, 128), (6, 2, 64), (9, 1, 128), (5, 5, 32), (4, 1, 96), (6, 2, 256), (16, 1, 64), (3, 1, 160)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 48])
def test_attention_of_single_tokens(dtype, heads, page):
    nq, nkv, d = heads
    lengths = [1, 2, 15, 16, 17, 31, 33, 64, 65, 130, 257]
    check(case(lengths, [1] * len(lengths), nq, nkv, d, page, dtype, seed=nq + d, spare_rows=2))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", HEADS)
def test_attention_of_prompts_and_mixed_steps(dtype, heads):
    nq, nkv, d = heads
    lengths, new = [37, 1, 90, 64, 5, 130, 20, 3], [37, 1, 33, 64, 2, 1, 19, 3]
    check(case(lengths, new, nq, nkv, d, 16, dtype, seed=nq + d, spare_rows=1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100, 1000])
@pytest.mark.parametrize("heads", [(4, 2, 128), (6, 2, 64), (2, 1, 96)])
def test_attention_in_a_window(dtype, window, heads):
    nq, nkv, d = heads
    lengths, new = [37, 1, 90, 150, 50, 131], [37, 1, 33, 1, 1, 140 - 9]
    c = case(lengths, new, nq, nkv, d, 16, dtype, window=window, seed=window + d)
    for r, (n, fresh) in enumerate(zip(lengths, new)):               # pages that a window has passed are given back
        for i in range(max(0, n - fresh - window + 1) // 16):
            c["table"][r][i] = -1
    check(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 96])
def test_attention_of_long_contexts(dtype, d):
    check(case([2049, 777, 1], [1, 1, 1], 4, 2, d, 16, dtype, seed=d))
    check(case([4097], [1], 4, 2, d, 32, dtype, seed=d))
    check(case([900, 411], [5, 140], 4, 2, d, 16, dtype, seed=d))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("new", [1, 20])
def test_pages_that_are_none_rows_without_keys_and_empty_requests(dtype, d, new):
    n = max(new, 1)
    c = case([70, 50, 40, n, 90], [n, n, 0, n, n], 4, 2, d, 16, dtype, seed=4,
             holes=[(0, 1, -1), (1, 0, 10 ** 6), (3, 0, -1), (3, 1, -1)] + [(4, i, -1) for i in range(6)])
    check(c)
    # a request that is shorter than what it brings: the rows in front of its first token see nothing
    c = case([3, 64], [n, n], 4, 2, d, 16, dtype, seed=4)
    check(c)
    # a sequence that is longer than its row of the table: the keys behind it are left out
    c = case([70, 33], [n, n], 4, 2, d, 16, dtype, seed=5)
    c["table"] = [row[:2] for row in c["table"]]
    check(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 32])
@pytest.mark.parametrize("new", [1, 9])
def test_what_lies_behind_the_last_token_is_not_read(dtype, d, new):
    """Stale words (not numbers among them) behind a sequence's end and before its window change nothing."""
    for window in (0, 20):
        c = case([21, 40, 64 + new], [new, new, new], 4, 2, d, 16, dtype, window=window, seed=8)
        first = attend(c).clone()
        places = np.array(P4._places(d))
        dirty = c["cache"].cpu().numpy()
        for r, n in enumerate(c["lengths"]):
            last = [j for j in range(n, (n + 15) // 16 * 16)]
            gone = list(range(0, max(0, n - new - window + 1))) if window else []
            for j in last + gone:
                m = dirty[c["table"][r][j // 16], :, 0]
                for plane in (0, 1):
                    word = places[j % 16, :, plane, 2]
                    m[:, word], m[:, word + 1] = 0xF0, 0x7F
        c["cache"] = torch.from_numpy(dirty).to(DEV)
        assert torch.equal(attend(c, torch.full_like(first, 5.0)), first)


@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("new", [1, 40])
def test_a_key_or_value_that_is_no_number_reaches_its_rows(d, new):
    c = case([60, 60], [new, new], 4, 2, d, 16, BF16, seed=2)
    clean = attend(c).clone()
    raw = c["cache"].cpu().numpy()
    places = np.array(P4._places(d))
    block = raw[c["table"][0][0], 0, 0]                              # request 0, kv head 0, token 3: its values 0..31
    at = places[3, 0, 1, 2]
    block[at], block[at + 1] = 0xF0, 0x7F
    block = raw[c["table"][1][0], 1, 0]                              # request 1, kv head 1, token 5: its keys 32..63
    at = places[5, 40, 0, 2]
    block[at], block[at + 1] = 0xF0, 0x7F
    c["cache"] = torch.from_numpy(raw).to(DEV)
    got = attend(c, torch.full_like(clean, 5.0)).reshape(2, new, 2, 2, d)
    clean = clean.reshape(2, new, 2, 2, d)
    assert torch.isnan(got[0, :, 0, :, :32]).all() and torch.equal(got[0, :, 0, :, 32:], clean[0, :, 0, :, 32:])
    assert torch.equal(got[0, :, 1], clean[0, :, 1]) and torch.equal(got[1, :, 0], clean[1, :, 0])
    assert torch.isnan(got[1, :, 1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 30])
def test_one_visible_key_gives_its_value(dtype, new):
    """A weight of one is not rounded: the result is what the cache holds."""
    c = case([50, 90], [new, new], 4, 2, 128, 16, dtype, window=1, seed=1)
    out = attend(c)
    _, values = P4.unpack(c["cache"], 128)
    for r in range(2):
        for i in range(new):
            j = c["lengths"][r] - new + i
            want = values[c["table"][r][j // 16], :, j % 16]
            got = out[c["starts"][r] + i].double().cpu().reshape(2, 2, 128)
            assert torch.equal(got[:, 0], want) and torch.equal(got[:, 1], want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores_do_not_overflow(dtype):
    c = case([200, 77], [1, 60], 4, 2, 128, 16, dtype, seed=6, sharp=300.0)
    out = attend(c)
    assert torch.isfinite(out).all()
    values = P4.unpack(c["cache"], 128)[1]
    assert float(out.abs().max()) <= float(values.abs().max()) * (1 + 2.0 ** -7)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB with a request in its last pages."""
    nkv, d, page = 8, 128, 16
    pages = (1 << 32) // (nkv * 18 * d) + 2000
    small = case([1000, 333], [1, 1], 16, nkv, d, page, BF16, seed=3)
    mixed = case([1000, 333], [1, 40], 16, nkv, d, page, BF16, seed=3)
    cache = torch.empty(kernels.kv4_cache_shape(pages, nkv, page, d), dtype=torch.uint8, device=DEV)
    shift = pages - small["cache"].shape[0]
    cache[shift:] = small["cache"]
    for c in (small, mixed):
        want = attend(c)
        c["cache"] = cache
        table = ints([[p + shift if p >= 0 else -1 for p in row] for row in c["table"]])
        assert torch.equal(attend(c, torch.empty_like(want), table=table), want)
    rows = rand(5, 32 * d, seed=4, dtype=BF16).to(DEV)
    slots = ints([pages * page - 1 - 3 * i for i in range(5)])
    kernels.qk_norm_rope_kv4_write(rows, ints([0] * 5), slots, None, None, 0.0, None, 0, cache, 16, nkv, d)
    keys, values = torch.empty(5, nkv * d, dtype=BF16, device=DEV), torch.empty(5, nkv * d, dtype=BF16, device=DEV)
    kernels.kv4_read(cache, slots, keys, values, nkv, d)
    assert float((values - rows[:, 24 * d:]).abs().max()) < 0.5


def test_other_streams_a_captured_graph_and_bounds_for_the_launch():
    c = case([300, 90, 41, 513], [1, 1, 20, 3], 8, 2, 128, 16, BF16, seed=9)
    want = attend(c).clone()
    # bounds instead of the numbers themselves, as a recorded step has them
    out = attend(c, torch.full_like(want, 5.0), longest=4000, lens=[25 + 128, 1, 1, 1])
    check(c, out)
    side = torch.cuda.Stream()
    args = (ints(c["table"]), ints(c["starts"]), ints(c["lengths"]))
    torch.cuda.synchronize()
    outs = [torch.empty_like(want) for _ in range(6)]
    for i in range(6):                                               # two streams at once
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            kernels.paged_attention_kv4(c["q"], outs[i], c["cache"], *args, c["new"], 8, 2, 128, c["scale"], max_seq_len=513)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for longest in (513, 2000):
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kernels.paged_attention_kv4(c["q"], out, c["cache"], *args, c["new"], 8, 2, 128, c["scale"], max_seq_len=longest)
        graphs.append((graph, out))
    for graph, out in graphs + graphs:
        out.fill_(9.0)
        graph.replay()
        check(c, out)
    c["lengths"] = [310, 20, 25, 7]                                  # the same graphs with shorter sequences
    args[2].copy_(ints(c["lengths"]))
    for graph, out in graphs:
        out.fill_(9.0)
        graph.replay()
        check(c, out)


def test_the_same_call_gives_the_same_bits():
    c = case([3000, 90, 1500], [1, 1, 1], 8, 2, 128, 16, BF16, seed=9)
    first = attend(c).clone()
    for _ in range(5):
        assert torch.equal(attend(c, torch.empty_like(first)), first)


# ---- the engine ------------------------------------------------------------------------------------------------------------

def engine_against_plain(model_folders, name, dtype, lengths, cut, tmp_path, monkeypatch, graphs=False):
    """Replays a trace on a cache of 4 bits.  The plain model then attends over the keys and values that the engine's cache holds
    (which it checks against its own: within half a step and the tolerance of the dtype)."""
    from cuinfer_b200.engine.runner import ModelRunner
    folders, cfg, block = model_folders[name]
    folder = folders[dtype]
    requests = {f"r{i}": random_tokens(cfg["vocab_size"], n, 700 + i) for i, n in enumerate(lengths)}
    steps = cut(requests)
    from cuinfer_b200.engine.replay import make_runner
    from cuinfer_b200.engine.runner import StepEntry
    monkeypatch.setattr(ModelRunner, "STEP_GRAPH_MIN_TOKENS", 2)
    runner = make_runner(folder, dtype, traces.live_token_peak(steps), block, max_live=max(4, len(requests)), cuda_graph=graphs, kv_cache_dtype="int4")
    nkv, d = cfg["num_key_value_heads"], cfg["head_dim"]
    held, logits = {}, {}
    for _ in range(3 if graphs else 1):
        for st in steps:
            entries = [StepEntry(e["id"], e["tokens"], e["want"]) for e in st["entries"]]
            at = {e.request_id: runner.manager.num_tokens(e.request_id) if e.request_id in runner.manager else 0 for e in entries}
            for e in entries:
                assert runner.reserve(e.request_id, len(e.tokens))
            if graphs and runner.can_use_graph(entries) and all(list(e.want) == [0] for e in entries):
                got = runner.decode_step(entries)
            else:
                got = runner.step(entries)
            got, row = got.float().cpu(), 0
            for e in entries:
                for w in e.want:
                    logits[e.request_id, at[e.request_id] + w] = got[row]
                    row += 1
            for rid in st.get("end", []):
                n = runner.manager.num_tokens(rid)
                slots = ints(runner.manager.slot_mapping(rid, 0, 0, n))
                for run in range(cfg["num_hidden_layers"]):
                    keys, values = (torch.empty(n, nkv * d, device=DEV) for _ in range(2))
                    kernels.kv4_read(runner.storage.run_cache[run], slots, keys, values, nkv, d)
                    held[rid, run] = (keys.cpu().view(n, nkv, d), values.cpu().view(n, nkv, d))
                runner.release(rid)
    kernels.check_error_flags(force=True)
    _, weights = P.load_folder(folder)
    plain = P.causal_attention
    worst = 0.0
    for rid, tokens in requests.items():
        layer = [0]

        def over_the_cache(q, k, v, scale, window=None):
            keys, values = held[rid, layer[0]]
            layer[0] += 1
            for mine, theirs in ((k, keys), (v, values)):
                span = mine.unflatten(-1, (-1, 32))
                half = 1.125 * (span.amax(-1).clamp(min=0) - span.amin(-1).clamp(max=0)) / 30
                slack = 3 * TOLERANCE[dtype] * float(mine.abs().max())
                assert ((mine - theirs).abs().unflatten(-1, (-1, 32)).amax(-1) <= half + slack).all()
            return plain(q, keys, values, scale, window)

        monkeypatch.setattr(P, "causal_attention", over_the_cache)
        want = P.forward(cfg, weights, tokens)
        monkeypatch.setattr(P, "causal_attention", plain)
        scale = float(want.abs().max())
        for i in range(len(tokens)):
            if (rid, i) in logits:
                worst = max(worst, float((logits[rid, i] - want[i]).abs().max()) / scale)
    assert worst <= TOLERANCE[dtype], f"{worst:.2e} of the largest logit"
    return runner


CUTS = {"whole": traces.whole, "tail": lambda r: traces.tail_decode(r, 24), "portions": traces.portions,
        "mixed": lambda r: traces.mixed(r, max_live=4)}


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "D"])
@pytest.mark.parametrize("cut", sorted(CUTS))
def test_engine(model_folders, name, dtype, cut, graphs, tmp_path, monkeypatch):
    engine_against_plain(model_folders, name, dtype, [40, 97, 130, 33], CUTS[cut], tmp_path, monkeypatch, graphs)


def test_generate_and_options(model_folders):
    from cuinfer_b200 import LLM, SamplingParams
    from cuinfer_b200.config import ConfigError
    folders, cfg, block = model_folders["D"]
    llm = LLM(folders["bfloat16"], block_size=block, num_blocks=64, max_num_seqs=8, kv_cache_dtype="int4")
    prompts = [random_tokens(cfg["vocab_size"], n, n) for n in (5, 60, 130)]
    greedy = SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True)
    first = [r.token_ids for r in llm.generate(prompts, greedy)]
    assert all(len(t) == 20 for t in first) and [r.token_ids for r in llm.generate(prompts, greedy)] == first
    plain = LLM(folders["bfloat16"], block_size=block, num_blocks=64, max_num_seqs=8)
    assert llm.engine.runner.page_bytes() * 32 == plain.engine.runner.page_bytes() * 9
    with pytest.raises(ConfigError, match="does not take a cache in 4 bits"):
        LLM(model_folders["A"][0]["bfloat16"], block_size=16, num_blocks=64, kv_cache_dtype="int4")       # head size 16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("window", [0, 24])
def test_a_later_value_that_is_no_number_does_not_reach_earlier_rows(dtype, d, window):
    """A key that a row does not see may hold a value or a key that is not a number: its weight is zero, and zero times that is not."""
    nq, nkv, lengths, new = 4, 2, [150, 90], [150, 70]
    c = case(lengths, new, nq, nkv, d, 16, dtype, window=window, seed=12)
    clean = attend(c).clone().reshape(-1, nkv, nq // nkv, d)
    raw = c["cache"].cpu().numpy()
    places = np.array(P4._places(d))
    spots = [(0, 70, 0, 1, 33), (0, 71, 1, 1, 3), (0, 140, 0, 1, 40), (1, 50, 0, 0, 5), (1, 88, 1, 1, 34)]         # request, token, kv head, plane, value
    for r, j, h, plane, i in spots:
        at = places[j % 16, i, plane, 2]
        block = raw[c["table"][r][j // 16], h, 0]
        block[at], block[at + 1] = 0xF0, 0x7F
    c["cache"] = torch.from_numpy(raw).to(DEV)
    got = attend(c, torch.full((sum(new), nq * d), 5.0, dtype=dtype, device=DEV)).reshape(-1, nkv, nq // nkv, d)
    for r, (n, fresh) in enumerate(zip(lengths, new)):
        for i in range(fresh):
            pos, row = n - fresh + i, c["starts"][r] + i
            for h in range(nkv):
                hit = torch.zeros(d, dtype=torch.bool)
                for rr, j, hh, plane, value in spots:
                    if rr == r and hh == h and j <= pos and (not window or j > pos - window):
                        if plane == 0:
                            hit[:] = True
                        else:
                            hit[value // 32 * 32:value // 32 * 32 + 32] = True
                bad = torch.isnan(got[row, h]).cpu()
                assert (bad == hit).all(), (r, i, h)
                assert torch.equal(got[row, h].cpu()[~bad], clean[row, h].cpu()[~bad]), (r, i, h)


@pytest.mark.parametrize("heads", [(2, 1, 128), (12, 4, 64), (5, 1, 128), (80, 2, 64), (8, 8, 128)])
@pytest.mark.parametrize("shape", ["one long", "many", "portions", "bounds"])
def test_prompts_of_many_row_tiles(heads, shape):
    nq, nkv, d = heads
    lengths, new = {"one long": ([700], [700]), "many": ([300, 270, 130, 257, 64, 65, 128, 129, 1, 2] * 2, [300, 270, 130, 257, 64, 65, 128, 129, 1, 2] * 2),
                    "portions": ([900, 64, 700, 300], [300, 64, 1, 129]), "bounds": ([257, 257, 257, 1, 30], [257, 257, 257, 1, 2])}[shape]
    if nq * sum(new) * max(lengths) > 12e6:
        lengths, new = [min(n, 130) for n in lengths], [min(n, 130) for n in new]
    c = case(lengths, new, nq, nkv, d, 16, BF16, seed=nq, spare_rows=3)
    if shape == "bounds":
        out = attend(c, lens=[sum(new) + 128] + [1] * (len(new) - 1), longest=5000)
        check(c, out)
    else:
        check(c)


def test_a_scale_that_is_not_positive():
    for scale in (0.0, -0.1):
        for new in (1, 40):
            c = case([90, 70], [new, new], 4, 2, 128, 16, BF16, seed=3)
            c["scale"] = scale
            check(c)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("shape", [(1, 0, 0), (2, 0, 0), (4, 0, 0), (8, 0, 0), (0, 5, 0), (0, 3, 8), (0, 64, 1), (0, 592, 8)])
def test_every_way_to_share_the_keys_of_single_tokens(monkeypatch, d, window, shape):
    """Clusters of every size, whole requests, and a list cut into any shares; among requests that bring several tokens or none."""
    monkeypatch.setattr(kernels, "kv4_decode_shape", lambda *args: shape)
    lengths, new = [700, 1, 33, 90, 410, 128, 0, 17, 259], [1, 1, 1, 40, 1, 1, 0, 1, 1]
    c = case(lengths, new, 6, 2, d, 16, BF16, window=window, seed=d, spare_rows=1)
    check(c)
    c = case([513, 0, 20], [1, 1, 1], 20, 2, d, 48, BF16, window=window, seed=d)
    check(c)


def test_how_the_keys_of_single_tokens_are_shared():
    assert kernels.kv4_decode_shape(8, 300, 592) == (4, 0, 0) and kernels.kv4_decode_shape(64, 4096, 592) == (8, 0, 0)
    assert kernels.kv4_decode_shape(8, 100, 592) == (1, 0, 0) and kernels.kv4_decode_shape(128, 4096, 592) == (4, 0, 0)
    assert kernels.kv4_decode_shape(512, 8192, 592) == (0, 592, 8) and kernels.kv4_decode_shape(32, 120001, 592) == (0, 592, 8)
    assert kernels.kv4_decode_shape(2000, 300, 592) == (0, 592, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("shares", [2, 3, 9])
def test_prompts_whose_keys_are_shared(monkeypatch, d, window, shares):
    monkeypatch.setattr(kernels, "kv4_prompt_shares", lambda *args: shares)
    check(case([700, 33, 1, 300, 64, 410], [130, 33, 1, 2, 64, 100], 4, 2, d, 16, BF16, window=window, seed=d + shares, spare_rows=2))
    # rows without keys, pages that are none, and bounds in the place of lengths
    c = case([3, 200, 90], [20, 20, 20], 6, 2, d, 16, BF16, window=window, seed=d, holes=[(1, i, -1) for i in range(13)] + [(2, 1, -1)])
    check(c)
    check(c, attend(c, torch.full_like(c["out"], 5.0), lens=[60 + 128, 1, 1], longest=900))


def test_a_value_that_is_no_number_in_one_share(monkeypatch):
    monkeypatch.setattr(kernels, "kv4_prompt_shares", lambda *args: 3)
    test_a_later_value_that_is_no_number_does_not_reach_earlier_rows(BF16, 128, 0)
    test_a_later_value_that_is_no_number_does_not_reach_earlier_rows(BF16, 64, 24)


def test_how_the_keys_of_prompts_are_shared():
    assert kernels.kv4_prompt_shares(128, 2048, 2048 * 2048) == 1 and kernels.kv4_prompt_shares(72, 4000, 1100 * 2048) == 2
    assert kernels.kv4_prompt_shares(8, 16384, 16 * 4096) == 18 and kernels.kv4_prompt_shares(8, 700, 16 * 4096) == 1
    assert kernels.kv4_prompt_shares(1, 120000, 4096 * 128) == 32


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [3, 1200])
@pytest.mark.parametrize("eps", [1e-6, 1e-36])
def test_keys_whose_squares_leave_the_range_of_32_bits(dtype, T, eps):
    """A row of 2^70 or 2^-70 times the others': its squares are infinite, or nothing, in 32 bits; its normed keys are like any others."""
    nq, nkv, d, page = 4, 2, 128, 16
    width = (nq + 2 * nkv) * d
    qkv = rand(T, width, seed=T, dtype=dtype)
    qkv[0, nq * d:(nq + nkv) * d] *= 2.0 ** 70
    qkv[1, nq * d:(nq + nkv) * d] *= 2.0 ** -70
    qkv[2, nq * d:(nq + nkv) * d] = 0.0
    gains = [(1 + rand(d, seed=s, scale=0.3)).to(dtype).to(DEV) for s in (1, 2)]
    table, positions = rope_table(600, d), torch.arange(T, dtype=torch.int32) % 600
    pages = (T + page - 1) // page
    cache = torch.zeros(kernels.kv4_cache_shape(pages, nkv, page, d), dtype=torch.uint8, device=DEV)
    kernels.qk_norm_rope_kv4_write(qkv.to(DEV), positions.to(DEV), ints(list(range(T))), *gains, eps, table, d, cache, nq, nkv, d)
    _, k, v = plain_rows(qkv, positions, *gains, eps, table, d, nq, nkv, d)
    at = torch.arange(T)
    for rows, hold in zip((k, v), P4.unpack(cache, d)):
        assert torch.equal(hold[at // page, :, at % page], torch.from_numpy(P4.held(rows.numpy().astype(np.float32))))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [128, 96])
@pytest.mark.parametrize("new", [1, 20])
def test_a_table_that_is_a_part_of_a_wider_one(dtype, d, new):
    """Keys behind the row's end have no page, whatever the memory behind the row holds."""
    c = case([70, 200, 50], [new] * 3, 4, 2, d, 16, dtype, seed=d + new)
    wide = ints([row[:6] + list(range(1, 9)) for row in c["table"]])
    c["table"] = [row[:6] for row in c["table"]]
    attend(c, table=wide[:, :6])
    check(c, c["out"])
    c["table"] = [row[2:6] for row in c["table"]]
    attend(c, table=wide[:, 2:6])
    check(c, c["out"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("cluster", [1, 2, 8])
def test_prompts_without_tensor_cores(monkeypatch, dtype, d, window, cluster):
    """Row tiles that end inside a request, a tile of a single row, single tokens among them, keys shared by none, a few or many."""
    monkeypatch.setattr(kernels, "kv4_rows_cluster", lambda *a: cluster)
    c = case([130, 1, 33, 300], [65, 1, 33, 1], 6, 2, d, 16, dtype, window=window, seed=d + cluster, spare_rows=2, holes=[(0, 1, -1), (3, 4, 99999)])
    if dtype == BF16:                                                # rows that are not 16-byte aligned: no tensor cores at any head size
        wide = torch.zeros(c["q"].shape[0], c["q"].shape[1] + 71, dtype=dtype, device=DEV)
        wide[:, 1:1 + c["q"].shape[1]] = c["q"]
        c["q"] = wide[:, 1:1 + c["q"].shape[1]]
    check(c)


@pytest.mark.parametrize("d", [96, 128])
@pytest.mark.parametrize("requests", [1, 3, 70])
def test_single_tokens_whose_keys_a_cluster_shares(d, requests):
    lengths = [1500, 260, 900][:requests] if requests < 4 else [(37 * r) % 700 for r in range(requests)]
    check(case(lengths, [1] * requests, 10, 2, d, 16, F32, seed=requests, holes=[(0, 0, -1)] if requests < 4 else ()))


def test_how_the_keys_of_row_tiles_are_shared():
    assert kernels.kv4_rows_cluster(1, 4000, 296) == 8 and kernels.kv4_rows_cluster(1, 128, 296) == 1
    assert kernels.kv4_rows_cluster(148, 4000, 296) == 2 and kernels.kv4_rows_cluster(149, 4000, 296) == 1
    assert kernels.kv4_rows_cluster(1, 257, 296) == 4


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("cluster", [1, 2, 8])
def test_prompts_of_head_sizes_between(monkeypatch, d, window, cluster):
    monkeypatch.setattr(kernels, "kv4_rows_cluster", lambda *a: cluster)
    check(case([130, 1, 33, 300], [65, 1, 33, 1], 6, 2, d, 16, BF16, window=window, seed=d + cluster, spare_rows=2, holes=[(0, 1, -1), (3, 4, 99999)]))
    check(case([400, 90], [31, 90], 9, 1, d, 48, BF16, window=window, seed=d, spare_rows=1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 96, 256])
def test_single_tokens_with_rows_behind_them_and_requests_without(dtype, d):
    """More rows than requests, and more requests than rows (as a padded step has): rows behind the last request stay."""
    check(case([40, 300, 17], [1, 1, 1], 4, 2, d, 16, dtype, seed=d, spare_rows=5))
    c = case([40, 300, 17, 0, 0], [1, 1, 1, 0, 0], 4, 2, d, 16, dtype, seed=d)
    check(c, attend(c, lens=[1] * 5))
