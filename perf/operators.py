# SPDX-License-Identifier: Apache-2.0
"""The operators of a decode step over a 4-bit paged key/value cache: their cases, their plain forms and their values in 64 bits.

Five operators, in the order in which a serving step calls them:

* ``plan``    block tables, slots and positions from request lengths (``ops.paging.plan_pages``)
* ``rope``    RMS norm of every query and key head and the position rotation in one pass (``ops.rope.qk_norm_rope``)
* ``bwd``     its gradients, for training (``ops.rope.qk_norm_rope_backward``)
* ``append``  keys and values into the 4-bit cache, alone or after norm and rotation, and back as the values they
              stand for (``ops.kv4.kv4_append``, ``kv4_append_rope``, ``kv4_read``)
* ``attn``    attention of ragged query rows over that cache (``ops.kv4.kv4_attention``)

The cache of one layer is a uint8 tensor [pages, kv heads, page / 16, 18 * D]: per block of 16 tokens the key codes
(16 * D / 2 bytes), the value codes, and for each token and 64 channels a bf16 scale and a bf16 midpoint of the keys,
then of the values.  value = midpoint + scale * (code - 7.5).
"""

import math
import random

import torch

own = False

GROUP = 64  # channels that share a scale and a midpoint


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # one generated token for each of 256 requests in flight, some of which end: what every serving step starts with
        {"name": "plan_decode_256", "op": "plan", "batch": 256, "page": 64, "width": 512, "low": 1, "high": 30000, "new": 1,
         "pad": 0, "ends": 16},
        # many short prompts admitted at once among running requests, with a padded batch
        {"name": "plan_prompts_2000", "op": "plan", "batch": 2000, "page": 16, "width": 300, "low": 0, "high": 4000, "new": 60,
         "pad": 777, "ends": 9},
        # the queries and keys of a small decode batch on one rank of eight
        {"name": "rope_decode_64_tp8", "op": "rope", "tokens": 64, "q_heads": 8, "kv_heads": 1, "dim": 128, "rot": 128,
         "norm": False, "inter": False, "dtype": "bfloat16"},
        # a long prompt with norms of queries and keys, all heads on one GPU
        {"name": "rope_prompt_8192", "op": "rope", "tokens": 8192, "q_heads": 64, "kv_heads": 8, "dim": 128, "rot": 128,
         "norm": True, "inter": False, "dtype": "bfloat16"},
        # the training step of one layer: gradients of queries, keys and both norms' weights
        {"name": "bwd_8192", "op": "bwd", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "norm": True,
         "inter": False, "dtype": "bfloat16"},
        # the same at an odd, small size: neighbouring pairs, half of the channels rotated
        {"name": "bwd_777_partial", "op": "bwd", "tokens": 777, "q_heads": 20, "kv_heads": 4, "dim": 64, "rot": 32,
         "norm": True, "inter": True, "dtype": "float16"},
        # a decode step's new keys and values: norm, rotation and the write in one call
        {"name": "append_decode_256", "op": "append", "tokens": 256, "q_heads": 64, "kv_heads": 8, "dim": 128, "rot": 128,
         "norm": True, "inter": False, "page": 64, "dtype": "bfloat16", "fused": True},
        # a prompt's keys and values, rotated before
        {"name": "append_prompt_16384", "op": "append", "tokens": 16384, "q_heads": 0, "kv_heads": 8, "dim": 128, "rot": 0,
         "norm": False, "inter": False, "page": 64, "dtype": "bfloat16", "fused": False},
        # one request on one rank of eight: latency
        {"name": "attn_decode_1x900_tp8", "op": "attn", "batch": 1, "low": 900, "high": 900, "q_low": 1, "q_high": 1,
         "q_heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "pad": 0, "idle": 0, "dtype": "bfloat16"},
        # a serving batch of ragged contexts: the cache's bytes
        {"name": "attn_decode_64_to_16k", "op": "attn", "batch": 64, "low": 500, "high": 16000, "q_low": 1, "q_high": 1,
         "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "pad": 0, "idle": 0, "dtype": "bfloat16"},
        # chunks of long prompts over what was cached before
        {"name": "attn_chunk_4x1024_to_9k", "op": "attn", "batch": 4, "low": 2000, "high": 9000, "q_low": 1024, "q_high": 1024,
         "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "pad": 0, "idle": 0, "dtype": "bfloat16"},
        # a few drafted tokens for each request, five query heads on one of keys, idle requests and padding
        {"name": "attn_verify_24_fp16", "op": "attn", "batch": 24, "low": 1, "high": 3000, "q_low": 1, "q_high": 5,
         "q_heads": 20, "kv_heads": 4, "dim": 64, "page": 16, "pad": 7, "idle": 7, "dtype": "float16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "bwd", "append", "attn", "attn"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "plan":
        batch = _spread(rng, 1, 2000)
        page = rng.choice([16, 32, 64, 128])
        width = _spread(rng, 8, 512 if batch <= 512 else 300)
        new = _spread(rng, 1, 200) if batch <= 512 else _spread(rng, 1, 60)
        new = min(new, page * width // 2)
        high = max(1, min(page * width - 2 * new, 60_000_000 // batch))
        return {"op": op, "batch": batch, "page": page, "width": width, "low": 0, "high": high, "new": new,
                "pad": rng.choice([0, 0, _spread(rng, 1, 1000)]), "ends": rng.choice([0, 3, 7, 16])}
    dim = rng.choice([64, 128, 128])
    if op in ("rope", "bwd"):
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        rot = rng.choice([dim, dim, 16 * rng.randint(1, dim // 16)])
        kv = rng.choice([1, 2, 4, 8])
        q = kv * rng.choice([1, 2, 4, 5, 8])
        most = 8192 * (72 if op == "rope" else 40) * 128 // ((q + kv) * dim)
        return {"op": op, "tokens": _spread(rng, 1, min(most, 40000)), "q_heads": q, "kv_heads": kv, "dim": dim, "rot": rot,
                "norm": rng.random() < 0.6 or op == "bwd", "inter": rng.random() < 0.3, "dtype": dtype}
    kv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        fused = rng.random() < 0.5
        q = kv * rng.choice([1, 4, 7, 8]) if fused else 0
        most = 16384 * 8 * 128 // (max(kv, (q + 2 * kv) // 3) * dim)
        return {"op": op, "tokens": _spread(rng, 1, min(most, 20000)), "q_heads": q, "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim // 2]) if fused else 0, "norm": fused and rng.random() < 0.6,
                "inter": fused and rng.random() < 0.3, "page": page, "dtype": dtype, "fused": fused}
    while True:
        group = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
        batch = _spread(rng, 1, 200)
        q_high = rng.choice([1, 1, 1, _spread(rng, 2, 8), _spread(rng, 9, 700)])
        high = _spread(rng, 1, 16000)
        case = {"op": "attn", "batch": batch, "low": rng.randint(0, high), "high": high, "q_low": rng.randint(1, q_high),
                "q_high": q_high, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "page": page,
                "pad": rng.choice([0, 0, _spread(rng, 1, 30)]), "idle": rng.choice([0, 0, 5]), "dtype": dtype}
        scores = batch * q_high * kv * group * high
        if scores <= 2.4e9 and batch * high * kv * dim <= 64 * 16000 * 8 * 128 and work(case)["flops"] <= 8e11:
            return case


def _ladder(n, low, high, turn):
    """n whole numbers from low to high in a ragged order that goes by the case alone."""
    return [low + int((i * 0.6180339887 + turn) % 1.0 * (high - low + 1)) for i in range(n)]


def _plan_lengths(c):
    lens = _ladder(c["batch"], c["low"], c["high"], 0.3)
    ends = [bool(c["ends"]) and i % c["ends"] == 3 for i in range(c["batch"])]
    # a prompt for one request in five, one token for the others; none for those that end
    new = [0 if e else c["new"] * 5 - 4 if c["new"] > 1 and i % 5 == 1 else 1 for i, e in enumerate(ends)]
    return lens, new, ends


def _attn_lengths(c):
    q = _ladder(c["batch"], c["q_low"], c["q_high"], 0.1)
    kv = _ladder(c["batch"], c["low"], c["high"], 0.5)
    if c["batch"] == 1:
        q, kv = [c["q_high"]], [c["high"]]
    for i in range(c["batch"]):
        if c["idle"] and i % c["idle"] == 2:
            q[i] = 0
        if kv[i]:  # the new tokens are cached before they attend; a request without a length has empty rows
            kv[i] = max(kv[i], q[i])
    return q, kv


def work(case):
    c = case
    if c["op"] == "plan":
        lens, new, ends = _plan_lengths(c)
        tokens = sum(new) + c["pad"]
        up = lambda n: -(-n // c["page"])  # noqa: E731
        freed = sum(up(n) for n, e in zip(lens, ends) if e)
        taken = sum(up(n + m) - up(n) for n, m, e in zip(lens, new, ends) if not e)
        touched = sum(up(n + m) - n // c["page"] for n, m, e in zip(lens, new, ends) if m)
        # lengths, new lengths and ends read; lengths, starts and page counts written; pages moved; three numbers a token
        return {"bytes": c["batch"] * (4 + 4 + 1 + 4 + 4 + 4) + 8 * freed + 8 * taken + 4 * touched + 12 * tokens, "flops": 0}
    size = 2
    if c["op"] in ("rope", "bwd"):
        rows = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        passes = 2 if c["op"] == "rope" else 3
        return {"bytes": passes * rows * c["dim"] * size + 4 * c["tokens"],
                "flops": rows * c["dim"] * (8 if c["op"] == "rope" else 16)}
    if c["op"] == "append":
        kv, q = c["tokens"] * c["kv_heads"] * c["dim"], c["tokens"] * c["q_heads"] * c["dim"]
        packed = 2 * kv * 9 // 16
        return {"bytes": 2 * kv * size + packed + packed + 2 * kv * size + 2 * q * size + 8 * c["tokens"],
                "flops": 2 * kv * 8 + (q + kv) * 8}
    q, kv = _attn_lengths(c)
    pairs = sum(sum(max(0, n - m + i + 1) for i in range(m)) for m, n in zip(q, kv))
    cached = sum(n for m, n in zip(q, kv) if m)
    rows = sum(q) + c["pad"]
    return {"bytes": cached * c["kv_heads"] * 2 * c["dim"] * 9 // 16 + 2 * rows * c["q_heads"] * c["dim"] * size
            + 4 * rows * c["q_heads"] + 4 * cached // c["page"],
            "flops": 4 * c["dim"] * c["q_heads"] * pairs}


# ---- the 4-bit blocks in plain torch -------------------------------------------

_LOW, _HIGH = [0, 4, 1, 5], [2, 6, 3, 7]  # which of 8 channels the low and the high half of each byte of a word hold


def _quantise(x):
    """[..., D] -> codes 0..15 (float), scale and midpoint [..., D / 64, 1], all in f32 with every step rounded once."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    # a quotient in 64 bits rounded to 32 is the correctly rounded one
    scale = ((high - low).double() / 15.0).float().bfloat16().float()
    mid = ((high + low) * 0.5).bfloat16().float()
    ratio = ((x - mid).double() / torch.where(scale > 0, scale, 1.0).double()).float()
    codes = (ratio + 7.5).round().clamp(0, 15)
    bad = ~(torch.isfinite(scale) & torch.isfinite(mid))
    scale, mid = torch.where(bad, math.nan, scale), torch.where(bad, math.nan, mid)
    return torch.where(bad, 0.0, codes).flatten(-2), scale, mid


def _words(codes, keys):
    """Codes [..., D] -> bytes [..., D / 2] in the cache's order of channels."""
    b = codes.to(torch.uint8).unflatten(-1, (-1, 8, 8))  # group, word, channel
    b = b[..., _LOW] | (b[..., _HIGH] << 4)
    if keys:  # pairs of words: pair, group, word of the pair
        return b.unflatten(-2, (4, 2)).movedim(-3, -4).flatten(-4)
    return b.movedim(-2, -3).flatten(-3)  # word, group


def _values(bytes_, scale, mid, keys):
    """The inverse, in f32: bytes [..., D / 2], scale and midpoint [..., D / 64] -> [..., D]."""
    g = scale.shape[-1]
    if keys:
        b = bytes_.unflatten(-1, (4, g, 2, 4)).movedim(-3, -4).flatten(-3, -2)
    else:
        b = bytes_.unflatten(-1, (8, g, 4)).movedim(-2, -3)
    codes = torch.empty(*b.shape[:-1], 8, dtype=torch.float32, device=b.device)
    codes[..., _LOW] = (b & 15).float()
    codes[..., _HIGH] = (b >> 4).float()
    return ((codes - 7.5) * scale[..., None, None] + mid[..., None, None]).flatten(-3)


def _row(offset, keys):
    """Where a token's codes stand in its block of 16: keys in order, values with the even ones of each eight first."""
    return offset if keys else (offset // 8) * 8 + (offset % 2) * 4 + offset % 8 // 2


def _params(scale, mid):
    return torch.stack([scale.squeeze(-1), mid.squeeze(-1)], -1).bfloat16().contiguous().view(torch.uint8).flatten(-2)


def _write(cache, k, v, slots):
    """Plain append: k, v [T, H, D] at slots (page * page size + place); negative slots are skipped."""
    pages, heads, blocks, _ = cache.shape
    dim = k.shape[-1]
    sent = slots.long()
    keep = (sent >= 0) & (sent < pages * blocks * 16)
    # skipped tokens are written to one spare block behind the cache
    flat = torch.cat([cache.movedim(1, 2).reshape(pages * blocks, heads, 18 * dim), cache.new_zeros(1, heads, 18 * dim)])
    block = torch.where(keep, sent // 16, pages * blocks)[:, None, None]
    head = torch.arange(heads, device=k.device)[None, :, None]
    at = (sent.clamp(min=0) % 16)[:, None, None]
    for x, keys, codes_at, params_at in ((k, True, 0, 16 * dim), (v, False, 8 * dim, 17 * dim)):
        codes, scale, mid = _quantise(x)
        n, m = dim // 2, dim // 16
        flat[block, head, codes_at + _row(at, keys) * n + torch.arange(n, device=k.device)] = _words(codes, keys)
        flat[block, head, params_at + at * m + torch.arange(m, device=k.device)] = _params(scale, mid)
    cache.copy_(flat[:-1].view(pages, blocks, heads, 18 * dim).movedim(2, 1))


def _read(cache, slots, dtype):
    pages, heads, blocks, width = cache.shape
    dim = width // 18
    sent = slots.long()
    keep = ((sent >= 0) & (sent < pages * blocks * 16))[:, None, None]
    sent = torch.where(keep[:, 0, 0], sent, 0)
    block = (sent // 16)[:, None, None]
    page, block = block // blocks, block % blocks
    head = torch.arange(heads, device=cache.device)[None, :, None]
    at = (sent % 16)[:, None, None]
    got = []
    for keys, codes_at, params_at in ((True, 0, 16 * dim), (False, 8 * dim, 17 * dim)):
        n, m = dim // 2, dim // 16
        codes = cache[page, head, block, codes_at + _row(at, keys) * n + torch.arange(n, device=cache.device)]
        p = cache[page, head, block, params_at + at * m + torch.arange(m, device=cache.device)]
        p = p.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
        got.append(torch.where(keep, _values(codes, p[..., 0], p[..., 1], keys), 0.0).to(dtype))
    return got


def _decode_blocks(cache):
    """[..., 18 * D] blocks -> keys and values [..., 16, D] in f32."""
    dim = cache.shape[-1] // 18
    got = []
    for keys, codes_at, params_at in ((True, 0, 16 * dim), (False, 8 * dim, 17 * dim)):
        codes = cache[..., codes_at:codes_at + 8 * dim].unflatten(-1, (16, dim // 2))
        codes = codes[..., _row(torch.arange(16, device=cache.device), keys), :]
        p = cache[..., params_at:params_at + dim].contiguous().view(torch.bfloat16).float().unflatten(-1, (16, -1, 2))
        got.append(_values(codes, p[..., 0], p[..., 1], keys))
    return got


# ---- plain forms -----------------------------------------------------------------


def _angles(positions, inv_freq):
    """cos and sin [T, 1, rot / 2]: the angle in 64 bits, since positions reach millions."""
    a = positions.double()[:, None, None] * inv_freq.double()
    return a.cos().float(), a.sin().float()


def _turn(x, cos, sin, inter, back=False):
    """Rotates the first 2 * cos.shape[-1] channels; back: by the negative angle."""
    half = cos.shape[-1]
    if back:
        sin = -sin
    head, tail = x[..., :2 * half], x[..., 2 * half:]
    a, b = (head[..., ::2], head[..., 1::2]) if inter else (head[..., :half], head[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([head, tail], -1)


def _norm_rope(x, weight, eps, cos, sin, inter):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.float()
    return _turn(y, cos, sin, inter).to(x.dtype)


def _norm_rope_back(dy, x, weight, eps, cos, sin, inter):
    g, xf = _turn(dy.float(), cos, sin, inter, back=True), x.float()
    if weight is None:
        return g.to(x.dtype), None
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps)
    n = xf * r
    dw = (g * n).double().sum((0, 1))
    g = g * weight.float()
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw.to(weight.dtype)


def _plain_plan(s):
    page, width = s["page"], s["table"].shape[1]
    old, new = s["lens"].long(), s["new"].long()
    left = torch.where(s["finished"], 0, old)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    have, want = (left + page - 1) // page, (left + new + page - 1) // page
    fits = (want <= width) & (starts[1:] <= s["tokens"])
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    released = torch.where(s["finished"], (old + page - 1) // page, 0)
    total = s["free_count"].long() + released.sum()
    granted = fits & ((need == 0) | (upto <= total))
    taken = torch.where(granted, upto, 0).amax()
    column = torch.arange(width, device=old.device)[None]
    # ended requests give their pages back on top of the stack, in order
    spare = s["free"].shape[0]
    goes = s["free_count"].long() + (released.cumsum(0) - released)[:, None] + column
    goes = torch.where(column < released[:, None], goes, spare)
    stack = torch.cat([s["free"], s["free"].new_zeros(1)]).scatter(0, goes.flatten(), s["table"].flatten())[:spare]
    # granted requests take theirs from its top
    comes = (total - taken + (upto - need)[:, None] + column - have[:, None]).clamp(0, spare - 1)
    mine = granted[:, None] & (column >= have[:, None]) & (column < want[:, None])
    table = torch.where(mine, stack[comes], s["table"])
    after = left + torch.where(granted, new, 0)
    t = torch.arange(s["tokens"], device=old.device)
    who = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    real = who < old.shape[0]
    who = who.clamp(max=old.shape[0] - 1)
    at = left[who] + t - starts[who]
    ok = real & granted[who]
    at = torch.where(ok, at, 0)
    slot = table[who, at // page].long() * page + at % page
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"positions": i32(at), "slots": i32(torch.where(ok, slot, -1)), "requests": i32(torch.where(real, who, -1)),
            "q_starts": i32(starts), "kv_lens": i32(torch.where(granted, after, 0)), "lens": i32(after),
            "free_count": i32(total - taken).reshape(1), "table": table, "free": stack}


def _plain_attention(q, cache, table, kv_lens, q_starts, q_most, kv_most):
    tokens, q_heads, dim = q.shape
    batch, heads = table.shape[0], cache.shape[1]
    page, group = cache.shape[2] * 16, q_heads // heads
    columns = max(1, -(-kv_most // page))
    k, v = _decode_blocks(cache[table[:, :columns].long().clamp(min=0)])  # batch, page, head, block, 16, dim
    k, v = (x.movedim(2, 1).flatten(2, 4) for x in (k, v))  # batch, head, key, dim
    key = torch.arange(k.shape[2], device=q.device)
    live = (key < kv_lens[:, None])[:, None, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    count = q_starts[1:] - q_starts[:-1]
    i = torch.arange(q_most, device=q.device)
    rows = (q_starts[:-1, None] + i).clamp(0, tokens - 1).long()
    x = q[rows].float().view(batch, q_most, heads, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (x @ k.transpose(-1, -2)).unflatten(2, (group, q_most)) * dim ** -0.5
    limit = (kv_lens - count)[:, None] + i + 1  # keys that query i of a request sees
    seen = (key < torch.minimum(limit, kv_lens[:, None])[..., None])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (group, q_most)) / torch.where(total == 0, 1.0, total)
    lse = (torch.log(total) + top).squeeze(-1)
    t = torch.arange(tokens, device=q.device)
    who = torch.searchsorted(q_starts[1:].contiguous(), t, right=True)
    real = who < batch
    who = who.clamp(max=batch - 1)
    at = (t - q_starts[who]).clamp(0, q_most - 1).long()
    o, lse = (y.permute(0, 3, 1, 2, *range(4, y.dim())).flatten(2, 3)[who, at] for y in (o, lse))
    return torch.where(real[:, None, None], o, 0.0).to(q.dtype), torch.where(real[:, None], lse, -math.inf)


# ---- inputs ------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _projected(c, g, tokens):
    """q, k and v as slices of one projection's output, keys with channels of larger size as models have them."""
    dtype, dim = getattr(torch, c["dtype"]), c["dim"]
    nq, nk = c["q_heads"], c["kv_heads"]
    x = torch.randn(tokens, nq + 2 * nk, dim, device="cuda", generator=g)
    x[:, nq:nq + nk] += 2.0 * torch.randn(dim, device="cuda", generator=g)
    x[:, nq:nq + nk, ::17] *= 4.0
    x = x.to(dtype)
    return x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:]


def _inv_freq(rot):
    return (500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def _rope_inputs(c, g):
    tokens, dtype = c["tokens"], getattr(torch, c["dtype"])
    q, k, v = _projected(c, g, tokens)
    start = int(torch.randint(0, 1_000_000, (1,), device="cuda", generator=g).item())
    weight = lambda: (1 + 0.2 * torch.randn(c["dim"], device="cuda", generator=g)).to(dtype)  # noqa: E731
    positions = (start + torch.arange(tokens, device="cuda")).to(torch.int32)
    return {"q": q, "k": k, "v": v, "positions": positions, "inv_freq": _inv_freq(c["rot"]) if c["rot"] else None,
            "q_weight": weight() if c["norm"] else None, "k_weight": weight() if c["norm"] else None, "eps": 1e-6,
            "inter": c["inter"]}


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "plan":
        lens, new, ends = _plan_lengths(c)
        page = c["page"]
        up = lambda n: -(-n // page)  # noqa: E731
        held = [up(n) for n in lens]
        taken = sum(up(n + m) - up(n) for n, m, e in zip(lens, new, ends) if not e)
        pages = sum(held) + taken + 50  # room for what this step asks for
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((c["batch"], c["width"]), -1, dtype=torch.int32, device="cuda")
        first = torch.tensor(held, device="cuda").cumsum(0) - torch.tensor(held, device="cuda")
        column = torch.arange(c["width"], device="cuda")[None]
        mine = column < torch.tensor(held, device="cuda")[:, None]
        table = torch.where(mine, order[(first[:, None] + column).clamp(max=pages - 1)], table)
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:pages - sum(held)] = order[sum(held):]
        return {"op": "plan", "lens": _ints(lens), "new": _ints(new), "finished": torch.tensor(ends, device="cuda"),
                "table": table, "free": free, "free_count": _ints([pages - sum(held)]), "page": page,
                "tokens": sum(new) + c["pad"]}
    if c["op"] in ("rope", "bwd"):
        s = {"op": c["op"], **_rope_inputs(c, g)}
        if c["op"] == "bwd":
            for name in ("q", "k"):
                s["d" + name] = torch.randn(s[name].shape, device="cuda", generator=g).to(s[name].dtype)
        return s
    if c["op"] == "append":
        s = {"op": "append", "fused": c["fused"], **_rope_inputs(c, g)}
        pages = -(-c["tokens"] // c["page"]) + 9
        s["slots"] = torch.randperm(pages * c["page"], device="cuda", generator=g)[:c["tokens"]].to(torch.int32)
        s["slots"][5::11] = -1  # rows of the padded batch
        s["cache"] = torch.randint(0, 256, (pages, c["kv_heads"], c["page"] // 16, 18 * c["dim"]), dtype=torch.uint8,
                                   device="cuda", generator=g)
        return s
    q_lens, kv_lens = _attn_lengths(c)
    dim, heads, page = c["dim"], c["kv_heads"], c["page"]
    held = [-(-n // page) for n in kv_lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((c["batch"], max(held) + 2), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor(held, device="cuda").cumsum(0) - torch.tensor(held, device="cuda")
    column = torch.arange(table.shape[1], device="cuda")[None]
    mine = column < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(mine, order[(first[:, None] + column).clamp(max=pages - 1)], table)
    cache = torch.empty(pages, heads, page // 16, 18 * dim, dtype=torch.uint8, device="cuda")
    # what no request holds is whatever the memory held before: here NaN in every scale
    live = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    key = torch.arange(table.shape[1] * page, device="cuda")[None]
    slot = table.long()[:, key[0] // page] * page + key % page
    live = torch.cat([live, live[:1]]).scatter(0, torch.where(key < _ints(kv_lens)[:, None], slot, pages * page).flatten(), True)
    live = live[:-1].view(pages, page // 16, 16)
    bias = 2.0 * torch.randn(heads, 1, 1, dim, device="cuda", generator=g)
    step = max(1, (1 << 27) // (heads * page * dim))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        for keys, codes_at, params_at in ((True, 0, 16 * dim), (False, 8 * dim, 17 * dim)):
            x = torch.randn(b - a, heads, page // 16, 16, dim, device="cuda", generator=g)
            if keys:
                x = x + bias
                x[..., ::17] *= 2.0
            codes, scale, mid = _quantise(x.bfloat16())
            dead = ~live[a:b, None, :, :, None, None]
            scale, mid = torch.where(dead, math.nan, scale), torch.where(dead, math.nan, mid)
            packed = torch.empty(b - a, heads, page // 16, 16, dim // 2, dtype=torch.uint8, device="cuda")
            packed[..., _row(torch.arange(16, device="cuda"), keys), :] = _words(codes, keys)
            cache[a:b, ..., codes_at:codes_at + 8 * dim] = packed.flatten(-2)
            cache[a:b, ..., params_at:params_at + dim] = _params(scale, mid).flatten(-2)
    rows = sum(q_lens) + c["pad"]
    q = torch.randn(max(rows, 1), c["q_heads"] + 2 * heads, dim, device="cuda", generator=g).to(getattr(torch, c["dtype"]))
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    return {"op": "attn", "q": q[:, :c["q_heads"]], "cache": cache, "table": table, "kv_lens": _ints(kv_lens),
            "q_starts": _ints(starts), "q_most": max(1, max(q_lens)), "kv_most": max(kv_lens)}


# ---- one pass --------------------------------------------------------------------------


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "plan":
        return _plain_plan(s)
    if s["op"] == "attn":
        out, lse = _plain_attention(s["q"], s["cache"], s["table"], s["kv_lens"], s["q_starts"], s["q_most"], s["kv_most"])
        return {"out": out, "lse": lse}
    if s["op"] == "append" and not s["fused"]:
        _write(s["cache"], s["k"], s["v"], s["slots"])
        k, v = _read(s["cache"], s["slots"], s["k"].dtype)
        return {"k": k, "v": v}
    cos, sin = _angles(s["positions"], s["inv_freq"])
    if s["op"] == "bwd":
        dq, dwq = _norm_rope_back(s["dq"], s["q"], s["q_weight"], s["eps"], cos, sin, s["inter"])
        dk, dwk = _norm_rope_back(s["dk"], s["k"], s["k_weight"], s["eps"], cos, sin, s["inter"])
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    q = _norm_rope(s["q"], s["q_weight"], s["eps"], cos, sin, s["inter"])
    k = _norm_rope(s["k"], s["k_weight"], s["eps"], cos, sin, s["inter"])
    if s["op"] == "rope":
        return {"q": q, "k": k}
    _write(s["cache"], k, s["v"], s["slots"])
    k, v = _read(s["cache"], s["slots"], k.dtype)
    return {"q": q, "k": k, "v": v}


def _run_own(s):
    if s["op"] == "plan":
        from vkccl_b200.ops.paging import plan_pages

        p = plan_pages(s["lens"], s["new"], s["table"], s["free"], s["free_count"], s["page"], s["tokens"],
                       finished=s["finished"])
        return {"positions": p.positions, "slots": p.slots, "requests": p.requests, "q_starts": p.q_starts,
                "kv_lens": p.kv_lens, "lens": p.lens, "free_count": p.free_count, "table": s["table"], "free": s["free"]}
    if s["op"] == "rope":
        from vkccl_b200.ops.rope import qk_norm_rope

        q, k = qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                            eps=s["eps"], interleaved=s["inter"])
        return {"q": q, "k": k}
    if s["op"] == "bwd":
        from vkccl_b200.ops.rope import qk_norm_rope_backward

        dq, dk, dwq, dwk = qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["positions"], s["inv_freq"],
                                                 q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"],
                                                 interleaved=s["inter"])
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    from vkccl_b200.ops.kv4 import kv4_append, kv4_append_rope, kv4_attention, kv4_read

    if s["op"] == "attn":
        out, lse = kv4_attention(s["q"], s["cache"], s["table"], s["kv_lens"], s["q_starts"], return_lse=True)
        return {"out": out, "lse": lse}
    got = {}
    if s["fused"]:
        got["q"] = kv4_append_rope(s["cache"], s["q"], s["k"], s["v"], s["slots"], s["positions"], s["inv_freq"],
                                   q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"], interleaved=s["inter"])
    else:
        kv4_append(s["cache"], s["k"], s["v"], s["slots"])
    got["k"], got["v"] = kv4_read(s["cache"], s["slots"], dtype=s["k"].dtype)
    return got


# ---- in 64 bits, from the definitions ------------------------------------------------------


def _complex_turn(x, positions, inv_freq, inter, sign):
    """The rotation as a product of complex numbers, in 64 bits."""
    half = inv_freq.shape[0]
    angle = sign * positions.double()[:, None] * inv_freq.double()[None]
    spin = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if inter else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., a], x[..., b]) * spin
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_norm(x, weight, eps):
    x = x.double()
    return x if weight is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def _exact_stored(x):
    """What 4 bits keep of x [T, H, D], in 64 bits."""
    got = torch.empty_like(x, dtype=torch.float64)
    for a in range(0, x.shape[-1], GROUP):
        y = x[..., a:a + GROUP].double()
        low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        scale, mid = ((high - low) / 15).bfloat16().double(), ((high + low) / 2).bfloat16().double()
        code = torch.clamp(torch.round((y - mid) / torch.where(scale == 0, 1.0, scale) + 7.5), 0, 15)
        got[..., a:a + GROUP] = mid + scale * (code - 7.5)
    return got


def _exact_cached(cache, pages, length):
    """Keys and values [heads, length, D] from the bytes of a request's pages, channel by channel, in 64 bits."""
    dim, heads = cache.shape[-1] // 18, cache.shape[1]
    raw = cache[pages].movedim(1, 0).reshape(heads, -1, 18 * dim)
    n, groups = raw.shape[1], dim // 64
    out = []
    for which in range(2):
        codes = raw[..., 8 * dim * which:8 * dim * (which + 1)].reshape(heads, n, 16, dim // 2)
        p = raw[..., 16 * dim + which * dim:17 * dim + which * dim].reshape(heads, n, 16, groups, 4).contiguous()
        p = p.view(torch.bfloat16).double()
        x = torch.empty(heads, n, 16, dim, dtype=torch.float64, device=cache.device)
        row = torch.tensor([t if which == 0 else 8 * (t // 8) + 4 * (t % 2) + (t % 8) // 2 for t in range(16)], device=cache.device)
        codes = codes[:, :, row]
        for d in range(dim):
            g, w, e = d // 64, d % 64 // 8, d % 8
            word = (w // 2) * 2 * groups + 2 * g + w % 2 if which == 0 else w * groups + g
            nibble = e // 2 + 4 * (e % 2)
            byte = codes[..., 4 * word + nibble // 2]
            code = (byte >> 4 if nibble % 2 else byte & 15).double()
            x[..., d] = p[..., g, 1] + p[..., g, 0] * (code - 7.5)
        out.append(x.reshape(heads, n * 16, dim)[:, :length])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "plan":
        return None  # whole numbers alone
    turn = lambda x, sign=1: _complex_turn(x, s["positions"], s["inv_freq"], s["inter"], sign)  # noqa: E731
    if op in ("rope", "append") and s["inv_freq"] is not None:
        q, k = (turn(_exact_norm(s[n], s[n + "_weight"], s["eps"])) for n in ("q", "k"))
        if op == "rope":
            return {"q": q, "k": k}
    if op == "append":
        k = k.to(s["k"].dtype) if s["fused"] else s["k"]  # rounded to the model's type, then to 4 bits
        got = {"q": q} if s["fused"] else {}
        keep = (s["slots"] >= 0)[:, None, None]
        got["k"], got["v"] = (torch.where(keep, _exact_stored(x), 0.0) for x in (k, s["v"]))
        return got
    if op == "bwd":
        got = {}
        for n in ("q", "k"):
            g, x, w = turn(s["d" + n].double(), -1), s[n].double(), s[n + "_weight"]
            if w is None:
                got["d" + n], got["dw" + n] = g, None
                continue
            size = (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
            got["dw" + n] = (g * x / size).sum((0, 1))
            gw = g * w.double()
            got["d" + n] = gw / size - x * (gw * x).mean(-1, keepdim=True) / size ** 3
        return got
    q, page = s["q"].double(), s["cache"].shape[2] * 16
    group = q.shape[1] // s["cache"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    starts, lens = s["q_starts"].tolist(), s["kv_lens"].tolist()
    for b, n in enumerate(lens):
        a, e = starts[b], starts[b + 1]
        if e == a or n == 0:
            continue
        pages = s["table"][b, :-(-n // page)].long()
        key, last = torch.arange(n, device="cuda"), n - (e - a) + torch.arange(e - a, device="cuda")
        hidden = key[None] > last[:, None]
        keys, values = _exact_cached(s["cache"], pages, n)
        for j in range(q.shape[1]):
            score = (q[a:e, j] @ keys[j // group].T / math.sqrt(q.shape[-1])).masked_fill(hidden, -math.inf)
            lse[a:e, j] = torch.logsumexp(score, -1)
            out[a:e, j] = torch.softmax(score, -1) @ values[j // group]
    return {"out": out, "lse": lse}
