"""The operators of the paged cache that is held in 4 bits, as they are measured: appending a step's keys and values (with
the norm and the rotation applied on the way), and attention over the cache.

A cache block holds 16 tokens of one key head in ``18 * D`` bytes: key codes, key words, value codes, value words.  A group is 32
neighbouring values of a head; its 16-bit word is a bfloat16 step with four significant bits whose low four bits hold the
zero point.  A value is ``step * (code - zero)``.
"""
import math
import random

import torch

own = False

GROUP = 32                     # values that share a word
BLOCK = 16                     # tokens of a cache block
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
POSITIONS = 4096               # rows of the rotation table at least
SMALLEST = 2.0 ** -120         # the smallest step


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    def write(name, dtype, tokens, heads, kv_heads, dim, rotary, norm, page):
        return {"name": name, "op": "write", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rotary, "norm": norm, "page": page}

    def attend(name, dtype, requests, context, new, singles, heads, kv_heads, dim, page, window, mix):
        return {"name": name, "op": "attend", "dtype": dtype, "requests": requests, "context": context, "new": new, "singles": singles,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "mix": mix}

    return [
        # a decode step of the benchmark's batch: eight tokens, each in a page of its own
        write("write_step_8", "bfloat16", 8, 16, 8, 128, 128, True, 16),
        # a prompt of the benchmark
        write("write_prompt_2048", "bfloat16", 2048, 16, 8, 128, 128, True, 16),
        # a whole token budget (8 192) less a few, at the larger sizes' heads
        write("write_prompt_8001", "bfloat16", 8001, 32, 8, 128, 128, True, 32),
        # a 32-bit model with a rotation of half the head and no norm
        write("write_f32_333", "float32", 333, 12, 3, 64, 32, False, 16),
        # one chat request that has just begun to answer
        attend("decode_1x300", "bfloat16", 1, 300, 1, 1, 16, 8, 128, 16, 0, 1),
        # the benchmark's decode step: batch 8 at 4 096 tokens
        attend("decode_8x4096", "bfloat16", 8, 4096, 1, 8, 16, 8, 128, 16, 0, 0),
        # a full server: 64 requests of any length up to 8 192, at the larger sizes' heads
        attend("decode_64x8192", "bfloat16", 64, 8192, 1, 64, 32, 8, 128, 16, 0, 2),
        # a few long documents
        attend("decode_4x120001", "bfloat16", 4, 120001, 1, 4, 32, 8, 128, 32, 0, 0),
        # a prompt of the benchmark
        attend("prompt_2048", "bfloat16", 1, 2048, 2048, 0, 16, 8, 128, 16, 0, 0),
        # a scheduler's mixed step: portions of three prompts beside 21 decoded tokens
        attend("mixed_24", "bfloat16", 24, 4000, 500, 21, 16, 8, 128, 16, 0, 3),
        # the last portion of a long prompt, at the larger sizes' heads
        attend("portion_2048_of_16384", "bfloat16", 1, 16384, 2048, 0, 32, 8, 128, 16, 0, 0),
        # a 32-bit model: a few short prompts
        attend("prompt_f32_3x211", "float32", 3, 211, 211, 0, 12, 3, 64, 16, 0, 4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        top = most.setdefault(case["op"], dict(w))
        for k in w:
            top[k] = max(top[k], w[k])
    while True:
        dtype = "float32" if rng.random() < 0.15 else "bfloat16"
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
        dim = rng.choice([64, 128, 128, 128]) if rng.random() < 0.8 else rng.choice([32, 96, 160, 256])
        page = rng.choice([16, 16, 16, 32, 48, 64])
        if rng.random() < 0.4:
            case = {"op": "write", "dtype": dtype, "tokens": _log(rng, 1, 8001), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                    "rotary": rng.choice([dim, dim, dim // 2, 0]), "norm": rng.random() < 0.6, "page": page}
        else:
            slow = dtype == "float32" or dim not in (64, 128)        # sizes of small models: short prompts and contexts
            kind = rng.choice(["decode", "decode", "prompt", "mixed"])
            requests = _log(rng, 1, 64) if kind == "decode" else _log(rng, 1, 24)
            context = _log(rng, 1, 4000 if slow else 120001 if kind == "decode" else 16384)
            new = 1 if kind == "decode" else min(context, _log(rng, 2, 400 if slow else 4096))
            singles = requests if kind == "decode" else rng.randrange(requests) if kind == "mixed" else 0
            window = rng.choice([0, 0, 0, max(1, context // 3)])
            case = {"op": "attend", "dtype": dtype, "requests": requests, "context": context, "new": new, "singles": singles, "heads": heads,
                    "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "mix": rng.randrange(1, 1000)}
            if requests * heads * new * context > 1 << 31:           # the plain form holds all scores at once
                continue
            if slow and work(case)["flops"] > 2e10:
                continue
        w = work(case)
        if all(w[k] <= most[case["op"]][k] for k in w):
            return case


def _lengths(case):
    """(tokens held after the step, tokens that the step brings) of every request.  ``mix`` 0: all as long as may be."""
    rng = random.Random(case["mix"])
    total, new = [], []
    for r in range(case["requests"]):
        n = 1 if r < case["singles"] else case["new"]
        length = case["context"]
        if case["mix"] and case["requests"] > 1:
            length = rng.randint(max(1, case["context"] // 8), case["context"])
            n = n if n == 1 else rng.randint(1, n)
        new.append(min(n, length))
        total.append(length)
    order = list(range(case["requests"]))
    if case["mix"]:
        rng.shuffle(order)
    return [total[i] for i in order], [new[i] for i in order]


def work(case):
    width = 2 if case["dtype"] == "bfloat16" else 4
    nq, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    held = nkv * d * 9 // 8                                  # bytes of a token's keys and values
    if case["op"] == "write":
        t = case["tokens"]
        # the rows, positions, slots and table rows in; queries, cache and the rows read back out
        return {"bytes": t * ((nq + 2 * nkv) * d * width + 8 + case["rotary"] * 4 + nq * d * width + held + held + 2 * nkv * d * width),
                "flops": t * ((nq + nkv) * (4 * d * case["norm"] + 3 * case["rotary"]) + 6 * nkv * d)}
    total, new = _lengths(case)
    pairs, read = 0, 0
    for length, n in zip(total, new):
        w = case["window"] or length
        pairs += sum(min(w, p + 1) for p in range(length - n, length))
        read += min(length, w + n - 1)
    return {"bytes": read * held + 2 * sum(new) * nq * d * width, "flops": 4 * pairs * nq * d}


# ---- the format in plain torch ---------------------------------------------------------------------------------------

def _quantise(x):
    """x float32 [..., D] -> (codes int32 [..., D], words int32 [..., D / 32])."""
    x = x.unflatten(-1, (-1, GROUP))
    bad = ~(x.abs() < 2.0 ** 127).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    low, high = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
    step = ((high - low) / torch.full_like(low, 15.0)).clamp(min=SMALLEST)               # (by a number it would be a product)
    step = ((step.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32)          # up to three bits behind the leading one
    zero = torch.round(-low / step)
    codes = (torch.round(x / step[..., None]) + zero[..., None]).clamp(0, 15).to(torch.int32)
    words = ((step.view(torch.int32) >> 16) & 0xFFF0) | zero.to(torch.int32)
    words = torch.where(bad, 0x7FF0, words)
    codes = torch.where(bad[..., None], 0, codes)
    return codes.flatten(-2), words


def _stands_for(codes, words):
    """The float32 values of codes [..., D] and words [..., D / 32]."""
    step = ((words & 0xFFF0) << 16).view(torch.float32)
    return ((codes.unflatten(-1, (-1, GROUP)) - (words & 15)[..., None]).float() * step[..., None]).flatten(-2)


def _as_bytes(x, size):
    return torch.stack([(x >> (8 * i)) & 255 for i in range(size)], -1).flatten(-2).to(torch.uint8)


def _pack(keys, values):
    """Blocks uint8 [..., 18 * D] of 16 tokens' float32 keys and values [..., 16, D]."""
    d = keys.shape[-1]
    groups = d // GROUP
    kc, kw = _quantise(keys)
    vc, vw = _quantise(values)
    shift = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=keys.device, dtype=torch.int64)
    k = kc.long().unflatten(-1, (groups, 4, 8))                            # token, group, quarter, value
    k = (k << shift).sum(-1).transpose(-1, -2).flatten(-3)                 # token, quarter, group
    v = vc.long().unflatten(-1, (groups, 8, 4)).unflatten(-4, (2, 4, 2))   # half, pair, token, group, eighth, value
    shift = torch.tensor([[4 * e + 16 * t for e in range(4)] for t in range(2)], device=keys.device, dtype=torch.int64)
    v = (v << shift[:, None, None, :]).sum(-1).sum(-3)                     # half, pair, group, eighth
    v = v.permute(*range(v.dim() - 3), -1, -3, -2).flatten(-4)             # half, eighth, pair, group
    vw = vw.unflatten(-2, (8, 2)).transpose(-1, -2).flatten(-3)            # pair, group, token
    return torch.cat([_as_bytes(k, 4), _as_bytes(kw.flatten(-2), 2), _as_bytes(v, 4), _as_bytes(vw, 2)], -1)


def _unpack(blocks, d):
    """float32 keys and values [..., 16, D] of blocks uint8 [..., 18 * D]."""
    groups = d // GROUP
    k, kw, v, vw = blocks.split([8 * d, d, 8 * d, d], -1)
    k = k.contiguous().view(torch.int32).unflatten(-1, (16, 4, groups)).transpose(-1, -2)
    shift = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=blocks.device, dtype=torch.int32)
    kc = ((k[..., None] >> shift) & 15).flatten(-3)
    kw = (kw.contiguous().view(torch.int16).to(torch.int32) & 0xFFFF).unflatten(-1, (16, groups))
    v = v.contiguous().view(torch.int32).unflatten(-1, (2, 8, 4, groups))
    v = v.permute(*range(v.dim() - 4), -4, -2, -1, -3)                     # half, pair, group, eighth
    shift = torch.tensor([[4 * e + 16 * t for e in range(4)] for t in range(2)], device=blocks.device, dtype=torch.int32)
    v = (v[..., None, :, :, None] >> shift[:, None, None, :]) & 15         # half, pair, token, group, eighth, value
    vc = v.flatten(-3).flatten(-4, -2)
    vw = (vw.contiguous().view(torch.int16).to(torch.int32) & 0xFFFF).unflatten(-1, (8, groups, 2)).transpose(-1, -2).flatten(-3, -2)
    return _stands_for(kc, kw), _stands_for(vc, vw)


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _rows(gen, rows, heads, dim):
    """Key-like rows: channels of unlike size, a few of them large, as projections of real inputs have."""
    size = torch.exp(0.4 * _normal(gen, 1, heads, dim))
    return _normal(gen, rows, heads, dim) * size + 0.5 * _normal(gen, 1, heads, dim) * size


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    dtype = TYPES[case["dtype"]]
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    state = {"op": case["op"], "heads": nq, "kv_heads": nkv, "dim": d, "page": page}
    blocks = page // BLOCK
    if case["op"] == "write":
        t = case["tokens"]
        rotary = case["rotary"]
        pages = (t + page - 1) // page + 3 if t > 64 else t + 3
        order = list(range(pages))
        rng.shuffle(order)
        if t > 64:                                    # a prompt's tokens fill page after page
            start = rng.randrange(page)
            slots = [order[(start + i) // page] * page + (start + i) % page for i in range(t)]
            positions = list(range(start, start + t))
        else:                                         # decoded tokens, each somewhere in a page of its own
            slots = [order[i] * page + rng.randrange(page) for i in range(t)]
            positions = [rng.randrange(POSITIONS) for _ in range(t)]
        rows = max(POSITIONS, t + page)
        state |= {
            "qkv": _rows(gen, t, nq + 2 * nkv, d).flatten(1).to(dtype), "rotary": rotary, "eps": 1e-6,
            "positions": torch.tensor(positions, dtype=torch.int32, device="cuda"), "slots": torch.tensor(slots, dtype=torch.int32, device="cuda"),
            "q_gain": (1.0 + 0.2 * _normal(gen, d)).to(dtype) if case["norm"] else None,
            "k_gain": (1.0 + 0.2 * _normal(gen, d)).to(dtype) if case["norm"] else None, "table": None,
            "cache": torch.zeros(pages, nkv, blocks, 18 * d, dtype=torch.uint8, device="cuda"),
        }
        if rotary:
            angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (
                -torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
            state["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        return state
    total, new = _lengths(case)
    need = [(n + page - 1) // page for n in total]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table, at = [], 0
    for length, n, count in zip(total, new, need):
        row = order[at:at + count]
        at += count
        if case["window"]:                            # pages that no query sees any more have been given back
            gone = max(0, length - n - case["window"] + 1) // page
            row = [-1] * gone + row[gone:]
        table.append(row + [-1] * (max(need) - count))
    cache = torch.empty(pages, nkv, blocks, 18 * d, dtype=torch.uint8, device="cuda")
    size = torch.exp(0.3 * _normal(gen, 2, nkv, 1, 1, d))
    for first in range(0, pages, 2048):               # (a part at a time: the numbers take eight times the cache's memory)
        part = cache[first:first + 2048]
        keys = _normal(gen, *part.shape[:3], BLOCK, d) * size[0]
        values = _normal(gen, *part.shape[:3], BLOCK, d) * size[1]
        part.copy_(_pack(keys, values))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state |= {
        # scores of a standard deviation of about two
        "q": (_rows(gen, starts[-1], nq, d) * 1.4).flatten(1).to(dtype), "cache": cache, "scale": d ** -0.5, "window": case["window"],
        "table": torch.tensor(table, dtype=torch.int32, device="cuda"),
        "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "lengths": torch.tensor(total, dtype=torch.int32, device="cuda"),
        "new": new, "longest": max(total),
    }
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------

def _plain_write(st):
    nq, nkv, d, page, rotary = st["heads"], st["kv_heads"], st["dim"], st["page"], st["rotary"]
    x = st["qkv"].unflatten(1, (-1, d))
    q, k, v = x[:, :nq].float(), x[:, nq:nq + nkv].double(), x[:, nq + nkv:].float()       # keys in 64 bits: values next to a border
    if st["q_gain"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + st["eps"]) * st["q_gain"].float()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + st["eps"]) * st["k_gain"].double()
    if rotary:
        cs = st["table"][st["positions"].long()][:, None]
        c, s, half = cs[..., 0], cs[..., 1], rotary // 2
        q = torch.cat([q[..., :half] * c - q[..., half:rotary] * s, q[..., half:rotary] * c + q[..., :half] * s, q[..., rotary:]], -1)
        c, s = c.double(), s.double()
        k = torch.cat([k[..., :half] * c - k[..., half:rotary] * s, k[..., half:rotary] * c + k[..., :half] * s, k[..., rotary:]], -1)
    slots = st["slots"].long()
    # the rows join what their blocks hold, and are read back from there
    blocks = st["cache"].shape[2]
    block = slots // page * blocks + slots % page // BLOCK
    held = st["cache"].transpose(1, 2).reshape(-1, nkv, 18 * d)
    mine, place = torch.unique(block, return_inverse=True)
    keys, values = _unpack(held[mine], d)
    keys[place, :, slots % BLOCK] = k.float()
    values[place, :, slots % BLOCK] = v
    held[mine] = _pack(keys, values)
    keys, values = _unpack(held[mine], d)
    kind = st["qkv"].dtype
    return {"q": q.flatten(1).to(kind), "keys": keys[place, :, slots % BLOCK].flatten(1).to(kind),
            "values": values[place, :, slots % BLOCK].flatten(1).to(kind)}


def _plain_attend(st):
    nq, nkv, d, page = st["heads"], st["kv_heads"], st["dim"], st["page"]
    g = nq // nkv
    table = st["table"].long()
    # every request's keys and values, [R, kv head, key, D]
    keys, values = _unpack(st["cache"][table.clamp(min=0)], d)
    keys, values = (x.permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for x in (keys, values))
    requests, held = table.shape[0], keys.shape[2]
    # queries padded to the longest portion, [R, kv head, head, token, D]
    starts, lengths = st["starts"].long(), st["lengths"].long()
    longest = max(st["new"])
    count = starts[1:] - starts[:-1]
    token = torch.arange(longest, device="cuda")
    live = token < count[:, None]
    row = (starts[:-1, None] + token).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][row].float().unflatten(-1, (nkv, g, d)).permute(0, 2, 3, 1, 4)
    scores = (q.flatten(2, 3) @ keys.transpose(-1, -2)).unflatten(2, (g, longest)) * st["scale"]
    key = torch.arange(held, device="cuda")
    position = ((lengths - count)[:, None] + token)[..., None]                        # [R, token, 1]
    seen = (key <= position) & live[..., None] & (table >= 0).repeat_interleave(page, 1)[:, None]
    if st["window"]:
        seen = seen & (key > position - st["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    values = values.masked_fill((key >= lengths[:, None])[:, None, :, None], 0.0)     # what no token has written yet may be anything
    out = (scores.flatten(2, 3) @ values).unflatten(2, (g, longest)) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).flatten(2)[live].to(st["q"].dtype)


def run(state):
    if own:
        from cuinfer_b200 import kernels
        nq, nkv, d = state["heads"], state["kv_heads"], state["dim"]
        if state["op"] == "write":
            qkv = state["qkv"]
            q = torch.empty(qkv.shape[0], nq * d, dtype=qkv.dtype, device=qkv.device)
            kernels.qk_norm_rope_kv4_write(qkv, state["positions"], state["slots"], state["q_gain"], state["k_gain"], state["eps"], state["table"],
                                           state["rotary"], state["cache"], nq, nkv, d, q_out=q)
            keys = torch.empty(qkv.shape[0], nkv * d, dtype=qkv.dtype, device=qkv.device)
            values = torch.empty_like(keys)
            kernels.kv4_read(state["cache"], state["slots"], keys, values, nkv, d)
            return {"q": q, "keys": keys, "values": values}
        out = torch.empty_like(state["q"])
        kernels.paged_attention_kv4(state["q"], out, state["cache"], state["table"], state["starts"], state["lengths"], state["new"],
                                    nq, nkv, d, state["scale"], state["window"], max_seq_len=state["longest"])
        return out
    return _plain_write(state) if state["op"] == "write" else _plain_attend(state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------------

def _held(numbers):
    """What float64 numbers [..., D] are held as."""
    x = numbers.reshape(*numbers.shape[:-1], numbers.shape[-1] // 32, 32)
    low = torch.minimum(x.min(-1, keepdim=True).values, torch.zeros((), dtype=torch.float64, device=x.device))
    high = torch.maximum(x.max(-1, keepdim=True).values, torch.zeros((), dtype=torch.float64, device=x.device))
    mantissa, exponent = torch.frexp(((high - low) / torch.full_like(low, 15)).clamp(min=2.0 ** -120))
    step = torch.ldexp(torch.ceil(mantissa * 16), exponent - 4)
    zero = torch.round(-low / step)
    code = torch.round(x / step + 0.0) + zero
    return (step * (code.clamp(0, 15) - zero)).reshape(numbers.shape)


def _exact_write(st):
    nq, nkv, d = st["heads"], st["kv_heads"], st["dim"]
    heads = st["qkv"].double().reshape(-1, nq + 2 * nkv, d)
    done = []
    for first, last, gain in ((0, nq, st["q_gain"]), (nq, nq + nkv, st["k_gain"])):
        x = heads[:, first:last].clone()
        if gain is not None:
            x = x * gain.double() * (x.pow(2).sum(-1, keepdim=True) / d + st["eps"]).pow(-0.5)
        half = st["rotary"] // 2
        for i in range(half):
            cos, sin = st["table"][st["positions"].long(), i].double().unbind(-1)
            a, b = x[..., i].clone(), x[..., i + half].clone()
            x[..., i] = a * cos[:, None] - b * sin[:, None]
            x[..., i + half] = b * cos[:, None] + a * sin[:, None]
        done.append(x)
    return {"q": done[0].flatten(1), "keys": _held(done[1].float().double()).flatten(1), "values": _held(heads[:, nq + nkv:]).flatten(1)}


def _numbers(block, d, plane):
    """float64 [tokens, D] of one plane of blocks uint8 [n, 18 * D], nibble by nibble."""
    byte = block[:, plane * 9 * d:(plane + 1) * 9 * d].long()
    groups = d // 32
    token = torch.arange(16, device=block.device)[:, None]
    value = torch.arange(d, device=block.device)[None, :]
    group, inside = value // 32, value % 32
    if plane == 0:
        bit = 32 * ((token * 4 + inside // 8) * groups + group) + 16 * (inside % 2) + 4 * (inside % 8 // 2)
        word = token * groups + group
    else:
        bit = 32 * (((token // 8 * 8 + inside // 4) * 4 + token % 8 // 2) * groups + group) + 16 * (token % 2) + 4 * (inside % 4)
        word = (token // 2 * groups + group) * 2 + token % 2
    code = (byte[:, bit // 8] >> (bit % 8)) & 15
    at = 8 * d + 2 * word
    word = byte[:, at] + 256 * byte[:, at + 1]
    power = torch.pow(2.0, ((word >> 7) - 127).double())
    step = power * (1 + ((word >> 4) & 7).double() / 8)
    return (step * (code - (word & 15))).reshape(-1, d)


def _exact_attend(st):
    nq, nkv, d, page = st["heads"], st["kv_heads"], st["dim"], st["page"]
    g = nq // nkv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, n in enumerate(st["new"]):
        length = int(st["lengths"][r])
        pages = st["table"][r, :(length + page - 1) // page].long()
        begin = 0
        if st["window"]:
            begin = max(0, length - n - st["window"] + 1) // page * page
        pages = pages[begin // page:]
        position = torch.arange(length - n, length, device="cuda").repeat_interleave(g)[:, None]
        at = torch.arange(begin, length, device="cuda")
        hidden = at > position
        if st["window"]:
            hidden = hidden | (at + st["window"] <= position)
        for h in range(nkv):
            block = st["cache"][pages, h].flatten(0, 1)
            keys, values = _numbers(block, d, 0)[:length - begin], _numbers(block, d, 1)[:length - begin]
            q = st["q"][first:first + n, h * g * d:(h + 1) * g * d].double().reshape(n * g, d)
            weights = torch.softmax((q @ keys.T * st["scale"]).masked_fill(hidden, -math.inf), -1)
            out[first:first + n, h * g * d:(h + 1) * g * d] = (weights @ values).reshape(n, g * d)
        first += n
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_write(state) if case["op"] == "write" else _exact_attend(state)
