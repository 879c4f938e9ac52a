# SPDX-License-Identifier: Apache-2.0
"""Plain implementations, in 64 bits or in whole numbers, that the tests of the
model operators (paging, rope, kv4) compare with."""

import math

import torch


def plan(lens, new, finished, table, free, count, page, tokens):
    """Page plan on python lists; returns a dict of what vcclPagePlan writes."""
    table, stack = [list(r) for r in table], list(free)
    top = count
    left = []
    for i, n in enumerate(lens):
        if finished[i]:
            for j in range(-(-n // page)):
                stack[top] = table[i][j]
                top += 1
        left.append(0 if finished[i] else n)
    starts, asked, grants, first, taken = [0], 0, [], [], 0
    for i, n in enumerate(new):
        n = max(n, 0)
        starts.append(starts[-1] + n)
        have, want = -(-left[i] // page), -(-(left[i] + n) // page)
        fits = want <= len(table[i]) and starts[-1] <= tokens
        need = want - have if fits else 0
        first.append(asked)
        asked += need
        ok = fits and (need == 0 or asked <= top)
        grants.append((ok, have, need))
        if ok and need:
            taken = asked
    bottom = top - taken
    kv, after = [], []
    for i, (ok, have, need) in enumerate(grants):
        if ok:
            for j in range(need):
                table[i][have + j] = stack[bottom + first[i] + j]
        kv.append(left[i] + max(new[i], 0) if ok else 0)
        after.append(left[i] + (max(new[i], 0) if ok else 0))
    pos, slots, who = [], [], [-1] * tokens
    for i in range(len(lens)):
        for t in range(starts[i], min(starts[i + 1], tokens)):
            who[t] = i
    for t, i in enumerate(who):
        if i >= 0 and grants[i][0]:
            p = left[i] + t - starts[i]
            pos.append(p)
            slots.append(table[i][p // page] * page + p % page)
        else:
            pos.append(0)
            slots.append(-1)
    return {"positions": pos, "slots": slots, "requests": who, "q_starts": starts, "kv_lens": kv, "lens": after,
            "free_count": [bottom], "table": table, "free": stack}


def spin(x, positions, inv_freq, interleaved, back=False):
    """Rotation in 64 bits."""
    half = inv_freq.shape[0]
    a = positions.double()[:, None, None] * inv_freq.double()
    c, s = a.cos(), a.sin() * (-1 if back else 1)
    y = x.clone()
    i = torch.arange(half, device=x.device)
    u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[..., u] = x[..., u] * c - x[..., v] * s
    y[..., v] = x[..., v] * c + x[..., u] * s
    return y


def norm_rope(x, weight, eps, positions, inv_freq, interleaved):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    return spin(x, positions, inv_freq, interleaved)


def stored(x):
    """Scale, midpoint and codes of every group of 64 channels, each step rounded once in f32 (on the CPU, whose
    f32 division is correctly rounded)."""
    x = x.detach().cpu().float().unflatten(-1, (-1, 64))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / torch.tensor(15.0)).bfloat16().float()
    m = ((hi + lo) * 0.5).bfloat16().float()
    codes = ((x - m) / torch.where(s > 0, s, torch.ones_like(s)) + 7.5).round().clamp(0, 15)
    bad = ~(torch.isfinite(s) & torch.isfinite(m))
    nan = torch.tensor(math.nan)
    return torch.where(bad, 0.0, codes), torch.where(bad, nan, s), torch.where(bad, nan, m)


def stored_values(x):
    codes, s, m = stored(x)
    return ((codes.double() - 7.5) * s.double() + m.double()).flatten(-2).to(x.device)


def attention(q, k, v, kv_lens, q_starts, scale):
    """q [T, Hq, D]; k, v: a list of [len, H, D] per request (f64).  Returns out, lse and, for a bound on the error,
    sum p |v| (the size of the terms that are added up)."""
    t, hq, d = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(kv_lens):
        a, e = q_starts[b], q_starts[b + 1]
        if e <= a or n == 0:
            continue
        group = hq // k[b].shape[1]
        kk, vv = (x.repeat_interleave(group, 1) for x in (k[b], v[b]))
        for i in range(a, e):
            see = max(0, n - (e - a) + (i - a) + 1)
            if not see:
                continue
            sc = torch.einsum("hd,nhd->hn", q[i].double(), kk[:see]) * scale
            p = torch.softmax(sc, -1)
            lse[i] = torch.logsumexp(sc, -1)
            out[i] = torch.einsum("hn,nhd->hd", p, vv[:see])
            size[i] = torch.einsum("hn,nhd->hd", p, vv[:see].abs())
    return out, lse, size
