"""Attention over the cache held in 4 bits in 64 bits, for tests only, with a bound of the arithmetic that the kernels do, element by
element: small enough that a key left out, a scale 1 % off or a result of fewer bits lies outside it.  Shares no code with
``cuinfer_b200``."""
from __future__ import annotations

import numpy as np
import torch

import plain_kv4 as P4


def planes(cache, d: int):
    """(step, code, zero) float64 [pages, nkv, page_size, d, 2 (keys, values)] of a cache tensor."""
    raw = cache.cpu().numpy().astype(np.int64)
    places = np.array(P4._places(d))
    code = (raw[..., places[..., 0]] >> places[..., 1]) & 15
    word = raw[..., places[..., 2]] + 256 * raw[..., places[..., 2] + 1]
    step = ((word & 0xFFF0) << 16).astype(np.uint32).view(np.float32).astype(np.float64)
    shape = (*raw.shape[:2], raw.shape[2] * 16, d, 2)
    return tuple(torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64).reshape(shape)) for x in (step, code, word & 15))


def attention(q, cache, block_table, starts, lengths, nq, nkv, d, scale, window=0, *, rounded, codes=False):
    """(out, allowed) float64 [T, nq, d].  ``rounded``: bfloat16 operands on tensor cores, else 32-bit multiply-adds throughout.  ``codes``: single
    tokens are computed from codes and zero points, whose products are larger than those of the numbers that they stand for.

    A score is off by its additions.  In 32 bits there are at most d + 8 roundings of 2^-24 of the sum of its terms' magnitudes S.  A
    tensor core adds 16 products and what it had, each cut at 2^-23 of the largest: 17 / 16 d + 8 of those for finished numbers (S = |scale| sum |q| |k|);
    from codes (S = |scale| sum |q| step (code + zero)) two products a group, 34, one product for the zero points, 17, a multiply-add a group and 18
    for the sums of q, the scale and the way back.  Going into the exponential it is rounded again, to 2^-23 of the row's largest S twice; the exponential is
    good to 2^-21.  So a weight p_j is off by a factor 1 + e_j, and the result by at most sum p_j e_j |v_j - out| / (1 - sum p_j e_j).

    The sums over N keys add N + 64 roundings of 2^-24 (17 / 16 N + 64 of 2^-23 on tensor cores) of sum p |v| + |out|: the denominator has as
    many.  With bfloat16 operands a weight (or a weight times a step) is rounded once for the numerator, 2^-8, and the result once more."""
    step, code, zero = planes(cache, d)
    number = step * (code - zero)
    keys, values, products = number[..., 0], number[..., 1], (step * (code + zero))[..., 0]
    pages, page, g, T = keys.shape[0], keys.shape[2], nq // nkv, q.shape[0]
    q = q.double().cpu()[:, :nq * d].reshape(T, nkv, g, d)
    out, allowed = torch.full((T, nkv, g, d), float("nan"), dtype=torch.float64), torch.zeros(T, nkv, g, d, dtype=torch.float64)
    unit = 2.0 ** -23 if rounded else 2.0 ** -24
    for r, length in enumerate(lengths):
        first, n = starts[r], starts[r + 1] - starts[r]
        if n == 0:
            continue
        index = torch.arange(length)
        column = index // page
        row = torch.tensor([int(x) for x in block_table[r]], dtype=torch.long)
        at = torch.where(column < len(row), row[column.clamp(max=len(row) - 1)], -1)
        named = (at >= 0) & (at < pages)
        at = torch.where(named, at, 0)
        position = torch.arange(length - n, length)[:, None]
        seen = named & (index <= position)
        if window:
            seen = seen & (index > position - window)
        from_codes = codes and rounded and n == 1
        adds = d + 8 if not rounded else 34 + 17 + d // 32 + 18 if from_codes else 17 * d / 16 + 8
        for h in range(nkv):
            k, v, c = keys[at, h, index % page], values[at, h, index % page], products[at, h, index % page]
            for a in range(g):
                x = q[first:first + n, h, a]
                s = (x @ k.T) * scale
                size = (x.abs() @ (c if from_codes else k.abs()).T) * abs(scale)
                size = torch.where(seen, size, 0.0)
                top = torch.where(seen, s, -torch.inf).amax(-1, keepdim=True) if length else s.sum(-1, keepdim=True)
                p = torch.where(seen, torch.exp(s - torch.where(top > -torch.inf, top, 0.0)), 0.0)
                p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
                o = p @ v
                e = torch.expm1((adds + 4) * unit * size + 2 * 2.0 ** -23 * (size.amax(-1, keepdim=True) if length else 0.0) + 2.0 ** -21)
                e = torch.where(seen, e, 0.0)
                # sum p e |v - o|, a column at a time: what is not seen has p = 0
                moved = torch.stack([((p * e) * (v[:, i] - o[:, i:i + 1]).abs()).sum(-1) for i in range(d)], -1)
                moved = moved / (1 - (p * e).sum(-1, keepdim=True)).clamp(min=1e-3)
                spread = p @ v.abs()
                count = seen.sum(-1, keepdim=True)
                extra = moved + ((count * 17 / 16 if rounded else count) + 64) * unit * (spread + o.abs())
                if rounded:
                    extra = extra + 2.0 ** -8 * 1.01 * spread
                    extra = extra + 2.0 ** -8 * (o.abs() + extra)
                out[first:first + n, h, a], allowed[first:first + n, h, a] = o, extra
    return out.reshape(T, nq, d), allowed.reshape(T, nq, d)


def worst(got, want, allowed, rows: int) -> float:
    """The largest share of what is allowed (infinite where a number is missing), over the first ``rows`` rows."""
    got = got.double().cpu().reshape(want.shape)[:rows]
    off = (got - want[:rows]).abs() / allowed[:rows].clamp(min=1e-30)
    return float("inf") if torch.isnan(off).any() else float(off.max()) if off.numel() else 0.0
