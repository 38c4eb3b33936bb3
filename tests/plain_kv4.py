"""The cache held in 4 bits, plain and slow, for tests only: the format value by value, and attention in 64 bits over what a
cache holds.  Shares no code with ``cuinfer_b200``."""
from __future__ import annotations

import numpy as np
import torch

F = np.float32


def quantise_group(x):
    """32 float32 values -> (codes, word), operation by operation in 32 bits."""
    x = np.asarray(x, dtype=np.float32)
    assert x.shape == (32,)
    if not all(abs(float(v)) < 2.0 ** 127 for v in x):
        return [0] * 32, 0x7FF0
    lo, hi = min(F(0), x.min()), max(F(0), x.max())
    t = max(F(F(hi - lo) / F(15)), F(2.0 ** -120))
    bits = int(t.view(np.uint32)) if hasattr(t, "view") else int(np.float32(t).view(np.uint32))
    bits = (bits + 0xFFFFF) & ~0xFFFFF
    step = np.array(bits, dtype=np.uint32).view(np.float32)[()]
    zero = int(np.rint(F(-lo / step)))
    codes = [min(15, max(0, int(np.rint(F(v / step))) + zero)) for v in x]
    return codes, (bits >> 16) | zero


def held(x):
    """What float32 values [..., d] are held as, float64: ``quantise_group`` for many groups at once."""
    x = np.asarray(x, dtype=np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    good = (np.abs(g) < F(2.0 ** 127)).all(-1, keepdims=True)
    g = np.where(good, g, F(0))
    lo, hi = np.minimum(g.min(-1, keepdims=True), F(0)), np.maximum(g.max(-1, keepdims=True), F(0))
    t = np.maximum((hi - lo) / F(15), F(2.0 ** -120))
    step = ((t.view(np.uint32) + np.uint32(0xFFFFF)) & ~np.uint32(0xFFFFF)).view(np.float32)
    zero = np.rint(-lo / step)
    code = np.clip(np.rint(g / step) + zero, 0, 15)
    out = step.astype(np.float64) * (code - zero).astype(np.float64)
    return np.where(good, out, np.nan).reshape(x.shape)


def value(code: int, word: int) -> float:
    """The number a code stands for (exact)."""
    step = float(np.array((word & 0xFFF0) << 16, dtype=np.uint32).view(np.float32)[()])
    return step * (code - (word & 15))


def _places(d: int):
    """For every (token, value index) of a block: where its codes and words of keys and values lie: (byte, shift, word byte) x 2."""
    groups = d // 32
    out = []
    for token in range(16):
        row = []
        for i in range(d):
            g, j = divmod(i, 32)
            quarter, e = divmod(j, 8)
            bit = 32 * ((token * 4 + quarter) * groups + g) + 4 * (e // 2) + 16 * (e % 2)
            key = (bit // 8, bit % 8, 8 * d + 2 * (token * groups + g))
            eighth, e = divmod(j, 4)
            bit = 32 * (((token // 8 * 8 + eighth) * 4 + token % 8 // 2) * groups + g) + 16 * (token % 2) + 4 * e
            row.append((key, (9 * d + bit // 8, bit % 8, 17 * d + 2 * ((token // 2 * groups + g) * 2 + token % 2))))
        out.append(row)
    return out


def read_block(block, d: int):
    """(keys, values) float64 [16, d] of one block's bytes."""
    block = np.asarray(block, dtype=np.int64)
    places = np.array(_places(d))                        # [16, d, 2, 3]
    code = (block[places[..., 0]] >> places[..., 1]) & 15
    word = block[places[..., 2]] + 256 * block[places[..., 2] + 1]
    step = (((word & 0xFFF0) << 16).astype(np.uint32)).view(np.float32).astype(np.float64)
    numbers = step * (code - (word & 15))
    return numbers[..., 0], numbers[..., 1]


def write_block(keys, values, d: int):
    """The bytes of a block of 16 tokens' float32 keys and values [16, d]."""
    block = np.zeros(18 * d, dtype=np.uint8)
    places = _places(d)
    for plane, rows in enumerate((keys, values)):
        for token in range(16):
            for g in range(d // 32):
                codes, word = quantise_group(rows[token][32 * g:32 * g + 32])
                for j, code in enumerate(codes):
                    byte, shift, at = places[token][32 * g + j][plane]
                    block[byte] |= code << shift
                block[at], block[at + 1] = word & 255, word >> 8
    return block


def unpack(cache, d: int):
    """keys, values float64 [pages, nkv, page_size, d] of a cache tensor (any device; on the CPU)."""
    raw = cache.cpu().numpy().astype(np.int64)
    places = np.array(_places(d))
    code = (raw[..., places[..., 0]] >> places[..., 1]) & 15
    word = raw[..., places[..., 2]] + 256 * raw[..., places[..., 2] + 1]
    step = (((word & 0xFFF0) << 16).astype(np.uint32)).view(np.float32).astype(np.float64)
    numbers = step * (code - (word & 15))                # [pages, nkv, blocks, 16, d, 2]
    numbers = numbers.reshape(*raw.shape[:2], raw.shape[2] * 16, d, 2)
    return torch.from_numpy(np.ascontiguousarray(numbers[..., 0])), torch.from_numpy(np.ascontiguousarray(numbers[..., 1]))


def attention(q, cache, block_table, starts, lengths, nq, nkv, d, scale, window=0, *, rounded=True, offset=True):
    """(out, allowed) float64 [T, nq, d]: attention in 64 bits, and how far a kernel may be off, element by element.

    A weight p and what it multiplies are off by the scores' error: a score is a sum of d products in 32 bits, of magnitudes
    |q| |k|, or |q| step (128 + 15) where the codes are multiplied with an offset of 128 (``offset``); each of its at most
    d + 8 additions is off by 2^-23 of the largest partial sum.  p = exp(score) takes that error, once in the weight and once in
    the denominator; the exponential itself is good to 2^-20.  With bfloat16 operands (``rounded``) p times the step is
    rounded once (2^-8) and the result once more (2^-8); rows of keys longer than 32 add N / 32 additions in 32 bits."""
    keys, values = unpack(cache, d)
    page = keys.shape[2]
    g = nq // nkv
    T = q.shape[0]
    q = q.double().cpu()[:, :nq * d].reshape(T, nq, d)
    out, allowed = torch.full((T, nq, d), float("nan"), dtype=torch.float64), torch.zeros(T, nq, d, dtype=torch.float64)
    for r, length in enumerate(lengths):
        n = starts[r + 1] - starts[r]
        where = [(int(block_table[r][j // page]), j % page) if j // page < len(block_table[r]) else (-1, 0) for j in range(length)]
        ok = torch.tensor([0 <= p < keys.shape[0] for p, _ in where], dtype=torch.bool)
        at = torch.tensor([p if 0 <= p < keys.shape[0] else 0 for p, _ in where], dtype=torch.long)
        off = torch.tensor([o for _, o in where], dtype=torch.long)
        for i in range(n):
            t, pos = starts[r] + i, length - n + i
            seen = ok.clone()
            index = torch.arange(length)
            seen &= index <= pos
            if window:
                seen &= index > pos - window
            for h in range(nkv):
                k, v = keys[at[seen], h, off[seen]], values[at[seen], h, off[seen]]
                for a in range(h * g, (h + 1) * g):
                    if not len(k):
                        out[t, a] = 0.0
                        continue
                    s = (k @ q[t, a]) * scale
                    p = torch.softmax(s, 0)
                    out[t, a] = p @ v
                    size = (k.abs() @ q[t, a].abs()).max()
                    if offset:                           # a step is at least the group's largest value / 15, and its range / 15 / 1.125
                        big = k.unflatten(-1, (-1, 32))
                        steps = 1.125 * (big.amax(-1).clamp(min=0) - big.amin(-1).clamp(max=0)).max(0).values / 7.0
                        size = (q[t, a].abs().unflatten(-1, (-1, 32)).sum(-1) * steps).sum() * 143
                    delta = (d + 8) * 2.0 ** -23 * abs(scale) * float(size) + 2.0 ** -20
                    spread = p @ v.abs()
                    sums = (len(k) / 32 + 64) * 2.0 ** -23
                    allowed[t, a] = spread * (2 * delta + sums + (2.0 ** -8 if rounded else 0.0)) * 1.02
                    if rounded:
                        allowed[t, a] += 2.0 ** -8 * (out[t, a].abs() + allowed[t, a])
    return out, allowed
