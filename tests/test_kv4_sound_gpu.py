"""The cache held in 4 bits on the GPU: calls that the first tests of it did not make."""
from __future__ import annotations

import random

import pytest
import torch

import plain_kv4_tight as tight
from cuinfer_b200 import kernels
from test_kv4_gpu import BF16, DEV, F32, attend, case

pytestmark = pytest.mark.gpu


def check(c, out=None, codes=True):
    """Against attention in 64 bits, within what the kernels' arithmetic may be off; rows behind the last request stay."""
    out = attend(c) if out is None else out
    kernels.check_error_flags(force=True)
    want, allowed = tight.attention(c["q"], c["cache"], c["table"], c["starts"], c["lengths"], c["nq"], c["nkv"], c["d"], c["scale"], c["window"],
                                    rounded=c["q"].dtype == BF16, codes=codes and c["d"] in (64, 128, 256))
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
