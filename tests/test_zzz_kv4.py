# SPDX-License-Identifier: Apache-2.0
"""The operators of a decode step over the 4-bit paged cache, against plain
implementations in 64 bits: page plan, norm + rotation and its gradients,
append / read, attention, and a run of them together."""

import math
import random

import pytest
import torch

import model_reference as ref
from conftest import gpu_count

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if gpu_count() == 0:
        pytest.skip("no GPU")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def inv_freq(rot, base=10000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, slack, what):
    """|got - want| <= slack everywhere, with the same NaN and infinities."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    d = (got - want).abs()[fine] - slack.expand_as(want)[fine]
    assert d.numel() == 0 or d.max().item() <= 0, (what, d.max().item())


# ---- plan ---------------------------------------------------------------------


def check_plan(lens, new, finished, table, free, count, page, tokens, **kw):
    from vkccl_b200.ops.paging import plan_pages

    want = ref.plan(lens, new, finished, table, free, count, page, tokens)
    d_table, d_free, d_lens, d_count = ints(table), ints(free), ints(lens), ints([count])
    p = plan_pages(d_lens, ints(new), d_table, d_free, d_count, page, tokens,
                   finished=torch.tensor(finished, device="cuda"), **kw)
    got = {n: getattr(p, n).tolist() for n in ("positions", "slots", "requests", "q_starts", "kv_lens", "lens", "free_count")}
    got["table"], got["free"] = d_table.tolist(), d_free.tolist()
    for n, x in want.items():
        assert got[n] == x, n
    assert d_lens.tolist() == lens and d_count.tolist() == [count]
    return got


def world(rng, batch, page, width, spare, most=None):
    """A consistent state: pages of the requests and the stack, all distinct."""
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, most or page * width)]) for _ in range(batch)]
    lens = [min(n, page * width) for n in lens]
    held = [-(-n // page) for n in lens]
    pages = list(range(sum(held) + spare))
    rng.shuffle(pages)
    table = [[-1] * width for _ in range(batch)]
    for i, h in enumerate(held):
        for j in range(h):
            table[i][j] = pages.pop()
    count = len(pages)
    return lens, table, pages + [-1] * sum(held), count


@pytest.mark.parametrize("seed", range(24))
def test_plan_matches_reference(seed):
    rng = random.Random(seed)
    batch, page, width = rng.choice([1, 2, 7, 40, 1030]), rng.choice([1, 3, 16, 64]), rng.choice([1, 5, 33])
    lens, table, free, count = world(rng, batch, page, width, rng.choice([0, 1, 5, 200]))
    if not free:
        free = [-1]
    new = [rng.choice([0, 0, 1, 1, 2, page, 3 * page + 1, -4]) for _ in range(batch)]
    finished = [rng.random() < 0.2 for _ in range(batch)]
    rows = sum(max(n, 0) for n in new)
    tokens = rng.choice([rows, rows + 9, max(rows - 2, 0)])
    check_plan(lens, new, finished, table, free, count, page, tokens)


def test_plan_largest_batch_and_empty():
    rng = random.Random(5)
    lens, table, free, count = world(rng, 8192, 16, 3, 9000, most=40)
    new = [i % 3 for i in range(8192)]
    check_plan(lens, new, [i % 5 == 0 for i in range(8192)], table, free, count, 16, sum(new) + 3)
    check_plan([0], [0], [False], [[7]], [3], 1, 16, 0)
    check_plan([5], [3], [True], [[7]], [3, 9], 1, 16, 3)  # ends and starts again in the same row


def test_plan_in_place_with_many_ends():
    """lens and free_count updated in place while other blocks still count the pages that ended requests give back."""
    from vkccl_b200.ops.paging import plan_pages

    rng = random.Random(9)
    for _ in range(20):
        lens, table, free, count = world(rng, 3000, 4, 40, 500)
        new = [rng.choice([0, 1, 9]) for _ in range(3000)]
        finished = [rng.random() < 0.5 for _ in range(3000)]
        want = ref.plan(lens, new, finished, table, free, count, 4, sum(new))
        d_lens, d_count, d_table, d_free = ints(lens), ints([count]), ints(table), ints(free)
        p = plan_pages(d_lens, ints(new), d_table, d_free, d_count, 4, sum(new), finished=torch.tensor(finished, device="cuda"),
                       lens_out=d_lens, count_out=d_count)
        assert d_lens.tolist() == want["lens"] and d_count.tolist() == want["free_count"] and d_free.tolist() == want["free"]
        assert d_table.tolist() == want["table"] and p.slots.tolist() == want["slots"]


def test_plan_refuses_in_order_and_returns_the_same_pages():
    # 4 pages free; asks 2, 3 (refused), 1 (behind it: refused), 0 (granted)
    got = check_plan([0, 0, 0, 3], [32, 48, 16, 2], [False] * 4, [[-1] * 4 for _ in range(3)] + [[9, -1, -1, -1]],
                     [1, 2, 3, 4], 4, 16, 98)
    assert got["kv_lens"] == [32, 0, 0, 5] and got["free_count"] == [2]
    # a step that releases what an equal step took gives the same pages back
    from vkccl_b200.ops.paging import plan_pages

    table, free = ints([[-1, -1], [-1, -1]]), ints([5, 6, 7, 8, 0, 0, 0, 0])
    lens, count, new = ints([0, 0]), ints([4]), ints([20, 9])
    plan_pages(lens, new, table, free, count, 16, 29, lens_out=lens, count_out=count)
    before = table.tolist()
    assert lens.tolist() == [20, 9] and count.tolist() == [1]
    plan_pages(lens, new, table, free, count, 16, 29, finished=torch.ones(2, dtype=torch.uint8, device="cuda"),
               lens_out=lens, count_out=count)
    assert table.tolist() == before and count.tolist() == [1]


def test_plan_corrupt_lengths_stay_in_bounds():
    """Lengths, counts and new lengths that no program should pass: nothing outside of the tensors is touched."""
    from vkccl_b200.ops.paging import plan_pages

    big = 2**31 - 1
    table, free = torch.full((3, 4), 1, dtype=torch.int32, device="cuda"), ints([2, 3, 4])
    p = plan_pages(ints([big, -7, 5]), ints([big, big, 1]), table, free, ints([big]), 16, 8,
                   finished=torch.tensor([True, False, False], device="cuda"))
    assert p.kv_lens.tolist() == [0, 0, 0] and p.requests.tolist() == [0] * 8  # int32 starts saturate
    p = plan_pages(ints([0, 0, 0]), ints([1, 1, 1]), table, free, ints([-5]), 16, 3)
    assert p.kv_lens.tolist() == [0, 0, 0] and p.free_count.tolist() == [0]


# ---- norm and rotation -------------------------------------------------------------


def rope_slack(want, dtype, size):
    """Half a step of the stored type, and f32 arithmetic: a dozen roundings of 2^-24 (norm, weight, cosines that are
    2^-23 off, products, sum) on terms of size `size` -> 2^-20."""
    return want.abs() * half_step(dtype) * (1 + 2**-6) + size * 2.0**-20 + 2.0**-25


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,rot,inter", [(128, 128, False), (128, 64, True), (64, 32, False), (80, 48, False),
                                           (96, 96, True), (256, 256, False), (192, 16, False), (16, 16, True)])
@pytest.mark.parametrize("tokens,hq,hk", [(1, 8, 1), (37, 5, 5), (700, 3, 1)])
def test_norm_rope_and_gradients(dtype, dim, rot, inter, tokens, hq, hk):
    from vkccl_b200.ops.rope import qk_norm_rope, qk_norm_rope_backward

    g = gen(dim + rot + tokens)
    qkv = randn(g, tokens, hq + 2 * hk, dim, dtype=dtype) * 3
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    pos, freq = ints([(i * 7919) % 2_000_000 for i in range(tokens)]), inv_freq(rot)
    for norm in (True, False):
        qw = (1 + 0.3 * randn(g, dim, dtype=dtype)) if norm else None
        kw = (1 + 0.3 * randn(g, dim, dtype=dtype)) if norm and inter else None  # one weight alone, too
        kw = kw if inter else qw
        yq, yk = qk_norm_rope(q, k, pos, freq, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=inter)
        for y, x, w, name in ((yq, q, qw, "q"), (yk, k, kw, "k")):
            want = ref.norm_rope(x, w, 1e-5, pos, freq, inter)
            close(y, want, rope_slack(want, dtype, want.abs().amax(-1, keepdim=True)), (name, norm))
        dyq, dyk = randn(g, tokens, hq, dim, dtype=dtype), randn(g, tokens, hk, dim, dtype=dtype)
        dq, dk, dwq, dwk = qk_norm_rope_backward(dyq, dyk, q, k, pos, freq, q_weight=qw, k_weight=kw, eps=1e-5,
                                                 interleaved=inter)
        for dx, dw, dy, x, w in ((dq, dwq, dyq, q, qw), (dk, dwk, dyk, k, kw)):
            leaf = x.double().detach().requires_grad_()
            wl = None if w is None else w.double().detach().requires_grad_()
            (ref.norm_rope(leaf, wl, 1e-5, pos, freq, inter) * dy.double()).sum().backward()
            size = leaf.grad.abs().amax(-1, keepdim=True)
            if w is not None:  # the projection term subtracts numbers of the size r |w g|
                size = size + (dy.double().abs().amax(-1, keepdim=True) * 4 * w.abs().max().double()
                               / (x.double().pow(2).mean(-1, keepdim=True) + 1e-5).sqrt())
            close(dx, leaf.grad, rope_slack(leaf.grad, dtype, size), "dx")
            assert (dw is None) == (w is None)
            if w is not None:
                # f32 sums of one lane's rows: at most rows * 2^-24 of the terms' sizes, each term 2^-20 off
                terms = (dy.double().abs().amax(-1) * 2 * math.sqrt(dim)).sum()
                close(dw, wl.grad, wl.grad.abs() * half_step(dtype) + terms * 2.0**-20 * (1 + tokens * 2.0**-4), "dw")


def test_gradients_against_differences():
    """Directional derivative of the f64 definition by central differences against the kernel's gradients."""
    from vkccl_b200.ops.rope import qk_norm_rope_backward

    g = gen(3)
    t, h, dim = 9, 3, 64
    q, k, w = randn(g, t, h, dim), randn(g, t, 1, dim), 1 + 0.2 * randn(g, dim)
    pos, freq = ints(list(range(t))), inv_freq(dim)
    dy, dyk = randn(g, t, h, dim), randn(g, t, 1, dim)
    dq, dk, dwq, dwk = qk_norm_rope_backward(dy, dyk, q, k, pos, freq, q_weight=w, k_weight=w)

    def loss(x, wt, d):
        return (ref.norm_rope(x, wt, 1e-6, pos, freq, False) * d.double()).sum()

    for x, d, dx, dw in ((q, dy, dq, dwq), (k, dyk, dk, dwk)):
        u, uw = torch.randn(x.shape, device="cuda", generator=g).double(), torch.randn(dim, device="cuda", generator=g).double()
        e = 1e-5
        num = (loss(x.double() + e * u, w.double(), d) - loss(x.double() - e * u, w.double(), d)) / (2 * e)
        ana = (dx.double() * u).sum()
        # each gradient is half a bf16 step off: independent errors of 2^-8 / sqrt(3) at most, 6 sigma
        assert abs(num - ana) <= 6 * 2.0**-8 * (dx.double() * u).pow(2).sum().sqrt() + 1e-6
        num = (loss(x.double(), w.double() + e * uw, d) - loss(x.double(), w.double() - e * uw, d)) / (2 * e)
        assert abs(num - (dw.double() * uw).sum()) <= 6 * 2.0**-8 * (dw.double() * uw).pow(2).sum().sqrt() + 1e-6


def test_norm_rope_in_place_strides_and_no_tokens():
    from vkccl_b200.ops.rope import qk_norm_rope, qk_norm_rope_backward

    g = gen(11)
    qkv = randn(g, 50, 7, 128)
    q, k, w = qkv[:, :4], qkv[:, 4:6], 1 + 0.1 * randn(g, 128)
    pos, freq = ints(list(range(50))), inv_freq(128)
    a, b = qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w)
    # heads first in memory, a broadcast input, outputs in place
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    ot = torch.empty(4, 50, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    a2, _ = qk_norm_rope(qt, k, pos, freq, q_weight=w, k_weight=w, q_out=ot)
    assert a2.data_ptr() == ot.data_ptr() and torch.equal(a, ot)
    e, _ = qk_norm_rope(q[:1].expand(50, 4, 128), k, pos, freq, q_weight=w, k_weight=w)
    e2, _ = qk_norm_rope(q[:1].repeat(50, 1, 1), k, pos, freq, q_weight=w, k_weight=w)
    assert torch.equal(e, e2)
    rest = qkv[:, 6].clone()
    qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(qkv[:, 6], rest)
    none = qkv[:0]
    a, b = qk_norm_rope(none[:, :4], none[:, 4:6], pos[:0], freq)
    assert a.shape == (0, 4, 128)
    out = qk_norm_rope_backward(none[:, :4], none[:, 4:6], none[:, :4], none[:, 4:6], pos[:0], freq, q_weight=w, k_weight=w)
    assert out[0].shape == (0, 4, 128) and out[2].abs().max() == 0 and out[3].abs().max() == 0


def test_backward_is_deterministic_and_rows_of_nan_stay_apart():
    from vkccl_b200.ops.rope import qk_norm_rope, qk_norm_rope_backward

    g = gen(12)
    q, k, w = randn(g, 3000, 4, 128), randn(g, 3000, 1, 128), 1 + 0.1 * randn(g, 128)
    dq, dk = randn(g, 3000, 4, 128), randn(g, 3000, 1, 128)
    pos, freq = ints(list(range(3000))), inv_freq(128)
    a = qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w)
    b = qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    y, _ = qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w)
    q[5, 2, 7], q[9, 0, 3] = math.nan, math.inf
    z, _ = qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w)
    keep = torch.ones(3000, 4, dtype=torch.bool, device="cuda")
    keep[5, 2] = keep[9, 0] = False
    assert torch.equal(z[keep], y[keep]) and torch.isnan(z[5, 2]).all()


# ---- append and read -------------------------------------------------------------


def unpack(block, dim, token, keys):
    """Codes, scales and midpoints of one token from a block's bytes, by the layout's definition."""
    raw = block.tolist()
    groups = dim // 64
    row = token if keys else (token & 8) + ((token & 1) << 2) + ((token & 7) >> 1)
    at = (0 if keys else 8 * dim) + row * (dim // 2)
    codes = []
    for d in range(dim):
        g, b, e = d // 64, d % 64 // 8, d % 8
        word = ((b >> 1) * groups + g) * 2 + (b & 1) if keys else b * groups + g
        nib = e // 2 + 4 * (e % 2)
        byte = raw[at + 4 * word + nib // 2]
        codes.append(byte >> 4 if nib % 2 else byte & 15)
    base = (16 if keys else 17) * dim + token * 4 * groups
    par = torch.tensor(raw[base:base + 4 * groups], dtype=torch.uint8).view(torch.bfloat16).view(groups, 2)
    return codes, par


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,page,hk", [(64, 16, 1), (128, 64, 3), (128, 48, 2)])
def test_append_bytes_and_read(dtype, dim, page, hk):
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_read

    g = gen(dim + page)
    t, pages = 90, 7
    kv = randn(g, t, 2 * hk, dim, dtype=dtype)
    kv[3] = 0.0                      # a constant group
    kv[4] = kv[4] * 1e-30 if dtype == torch.bfloat16 else kv[4] * 1e-4
    kv[5, :, 7] = 100.0
    kv[6, 0, 9] = math.nan
    kv[7, hk, dim - 1] = -math.inf
    kv[8] = (kv[8] > 0).to(dtype) * 15 - 7.5  # exact ties are not moved: codes 0 and 15
    kv[9] = torch.arange(dim, device="cuda").to(dtype) % 16
    k, v = kv[:, :hk], kv[:, hk:]
    cache = torch.randint(0, 256, kv4_alloc(pages, page, hk, dim).shape, dtype=torch.uint8, device="cuda", generator=g)
    before = cache.clone()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:t].int()
    slots[0], slots[1], slots[2] = -1, pages * page, 2**31 - 1
    kv4_append(cache, k, v, slots)
    got_k, got_v = kv4_read(cache, slots, dtype=torch.float32)
    for x, y in ((k, got_k), (v, got_v)):
        want = ref.stored_values(x)
        want[:3] = 0.0
        # one f32 rounding of the result
        close(y, want, want.abs() * 2.0**-23, "read")
        b, = kv4_read(cache, slots, dtype=dtype)[0 if y is got_k else 1:][:1]
        close(b, want, want.abs() * half_step(dtype) * (1 + 2**-10) + 2.0**-25, "read in 16 bits")
    # the bytes, by the layout's definition, for a few tokens
    codes, s, m = ref.stored(k)
    vcodes, vs, vm = ref.stored(v)
    for i in (3, 4, 5, 8, 9, 40, 89):
        p, o = divmod(int(slots[i]), page)
        for keys, (c, sc, mi) in ((True, (codes, s, m)), (False, (vcodes, vs, vm))):
            gc, gp = unpack(cache[p, hk - 1, o // 16].cpu(), dim, o % 16, keys)
            assert gc == c[i, hk - 1].flatten().int().tolist()
            assert torch.equal(gp[:, 0].float(), sc[i, hk - 1, :, 0]) and torch.equal(gp[:, 1].float(), mi[i, hk - 1, :, 0])
    # nothing else changed: undo the written tokens' bytes and compare
    touched = torch.zeros_like(cache, dtype=torch.bool)
    gcount = dim // 64
    for sl in slots.tolist():
        if not 0 <= sl < pages * page:
            continue
        p, o = divmod(sl, page)
        b, tk = o // 16, o % 16
        vr = (tk & 8) + ((tk & 1) << 2) + ((tk & 7) >> 1)
        for lo, n in ((tk * (dim // 2), dim // 2), (8 * dim + vr * (dim // 2), dim // 2), (16 * dim + tk * 4 * gcount, 4 * gcount),
                      (17 * dim + tk * 4 * gcount, 4 * gcount)):
            touched[p, :, b, lo:lo + n] = True
    assert torch.equal(torch.where(touched, before, cache), before)


@pytest.mark.parametrize("inter,norm,rot", [(False, True, 128), (True, False, 64), (False, False, 32)])
@pytest.mark.parametrize("tokens", [1, 200, 2500])
def test_append_rope_is_rope_then_append(inter, norm, rot, tokens):
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_append_rope
    from vkccl_b200.ops.rope import qk_norm_rope

    g = gen(tokens)
    qkv = randn(g, tokens, 8 + 2 * 2, 128)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    w = 1 + 0.1 * randn(g, 128) if norm else None
    pos, freq = ints([i * 3 for i in range(tokens)]), inv_freq(rot)
    slots = torch.randperm(tokens + 64, device="cuda", generator=g)[:tokens].int()
    a, b = (kv4_alloc(-(-(tokens + 64) // 32), 32, 2, 128) for _ in range(2))
    out = kv4_append_rope(a, q, k, v, slots, pos, freq, q_weight=w, k_weight=w, interleaved=inter)
    yq, yk = qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w, interleaved=inter)
    kv4_append(b, yk, v, slots)
    assert torch.equal(out, yq) and torch.equal(a, b)


def test_append_and_read_of_no_tokens():
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_read

    cache = kv4_alloc(1, 16, 1, 64)
    none = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    kv4_append(cache, none, none, ints([]))
    k, v = kv4_read(cache, ints([]))
    assert k.shape == (0, 1, 64) and cache.abs().max() == 0


# ---- attention -----------------------------------------------------------------------


def filled(g, kv_lens, page, hk, dim, extra_pages=2, dtype=torch.bfloat16, width=None, spread=1.0):
    """A cache with the requests' keys and values appended, NaN in everything else, and a shuffled table."""
    from vkccl_b200.ops.kv4 import kv4_append, kv4_alloc, kv4_read

    held = [-(-n // page) for n in kv_lens]
    pages = sum(held) + extra_pages
    cache = torch.full_like(kv4_alloc(pages, page, hk, dim), 255)
    order = torch.randperm(pages, device="cuda", generator=g).tolist()
    width = width or max(held + [1]) + 1
    table = [[-1] * width for _ in kv_lens]
    slots = []
    for i, n in enumerate(kv_lens):
        for j in range(held[i]):
            table[i][j] = order.pop()
        slots += [table[i][t // page] * page + t % page for t in range(n)]
    slots = ints(slots)
    kv = randn(g, len(slots), 2 * hk, dim, dtype=dtype)
    kv[:, :hk] += randn(g, 1, hk, dim, dtype=dtype) * 2
    kv = kv * (1 + spread * torch.rand(len(slots), 2 * hk, 1, device="cuda", generator=g)).to(dtype)
    kv4_append(cache, kv[:, :hk], kv[:, hk:], slots)
    k, v = kv4_read(cache, slots, dtype=torch.float32)
    ends = torch.tensor([0] + kv_lens).cumsum(0).tolist()
    ks, vs = ([x[a:b].double() for a, b in zip(ends, ends[1:])] for x in (k, v))
    return cache, ints(table), ks, vs


def check_attention(got, lse, q, ks, vs, kv_lens, q_starts, scale=None):
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    want, wlse, size = ref.attention(q, ks, vs, kv_lens, q_starts, scale)
    # The largest sum of absolute products behind a score: (7.5 scale + |mid|) bounds a value, and with it f32 keeps a
    # score to 2^-19 of it (products of exact codes, a handful of f32 roundings and 128 additions of 2^-24 each).
    most = [x.abs().amax() * 3 if x.numel() else torch.zeros((), dtype=torch.float64, device="cuda") for x in ks]
    big = torch.stack(most).max() if most else torch.zeros((), dtype=torch.float64, device="cuda")
    score = (q.double().abs().sum(-1) * big * abs(scale))[..., None] * 2.0**-19
    vmax = max([x.abs().max().item() for x in vs if x.numel()] + [0.0])
    n = max(kv_lens + [0])
    # weights rounded to f16 (2^-11 and its half step 2^-12, on codes up to 7.5 of a scale: 2 vmax covers them), their
    # subnormal end (2^-25 a token), scores, and the stored type
    slack = want.abs() * half_step(q.dtype) * (1 + 2**-6) + size * 2.0**-11 + vmax * 2.0**-11 * 2 * (1 / math.sqrt(max(n, 1)) + 2.0**-4) \
        + n * 2.0**-25 * vmax + (size + vmax * 2.0**-4) * score + 2.0**-25
    # Requests with many rows: scores are exact to f32 too; a value is o + s (code - 8) with o = mid + s / 2 rounded to f16
    # (|o| <= 1.1 max |v|) and the sum rounded, the weights are rounded: 2^-11 each of what they are.
    heads = ks[0].shape[1]
    long = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device="cuda")
    if q.shape[0] * (q.shape[1] // heads) >= 64:
        for a, e in zip(q_starts, q_starts[1:]):
            if (e - a) * (q.shape[1] // heads) >= 64:
                long[a:e] = 1.0
    slack = slack + long * 2.0**-11 * (2 * size + 1.1 * vmax)
    close(got, want, slack, "out")
    if lse is not None:
        close(lse, wlse, score[..., 0] + wlse.abs().nan_to_num(posinf=0) * 2.0**-20 + 2.0**-19, "lse")


def starts(q_lens):
    return [0] + torch.tensor(q_lens).cumsum(0).tolist()


LENS = [1, 0, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 300, 1000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,hk,group", [(16, 1, 8), (64, 2, 1), (32, 2, 4), (48, 1, 5), (64, 1, 16), (128, 3, 3), (16, 1, 20)])
def test_attention_single_tokens(dtype, dim, page, hk, group):
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(dim + page + group)
    cache, table, ks, vs = filled(g, LENS, page, hk, dim)
    qs = starts([1] * len(LENS))
    q = randn(g, len(LENS) + 3, hk * group, dim, dtype=dtype)
    out, lse = kv4_attention(q, cache, table, ints(LENS), ints(qs), return_lse=True)
    check_attention(out, lse, q, ks, vs, LENS, qs)
    assert out[len(LENS):].abs().max() == 0 and torch.isinf(lse[len(LENS):]).all()  # the padded batch
    again = kv4_attention(q, cache, table, ints(LENS), ints(qs))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dim,page,hk,group,dtype", [(128, 64, 2, 8, torch.bfloat16), (64, 16, 1, 5, torch.float16),
                                                     (128, 32, 1, 1, torch.float16), (128, 16, 2, 4, torch.bfloat16)])
@pytest.mark.parametrize("q_lens", [[2, 1, 0, 3, 8, 1], [40, 1, 17, 5, 129, 0], [300, 7, 256, 64, 33, 2]])
def test_attention_several_tokens(dim, page, hk, group, dtype, q_lens):
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(dim + page + sum(q_lens))
    kv_lens = [n + c if n else 20 for n, c in zip(q_lens, [0, 40, 0, 500, 61, 1])]
    kv_lens[1] = 0  # rows without a single key
    cache, table, ks, vs = filled(g, kv_lens, page, hk, dim)
    qs = starts(q_lens)
    q = randn(g, qs[-1], hk * group, dim, dtype=dtype)
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(qs), return_lse=True)
    check_attention(out, lse, q, ks, vs, kv_lens, qs)


def test_attention_more_rows_than_tokens():
    """A request with more rows than cached tokens: its first rows see nothing."""
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(4)
    kv_lens, q_lens = [5, 3], [9, 40]
    cache, table, ks, vs = filled(g, kv_lens, 16, 1, 128)
    q = randn(g, 49, 4, 128)
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(starts(q_lens)), return_lse=True)
    check_attention(out, lse, q, ks, vs, kv_lens, starts(q_lens))
    assert out[:4].abs().max() == 0 and torch.isinf(lse[:4]).all()


@pytest.mark.parametrize("kv,batch,group", [(5000, 3, 8), (20000, 1, 8), (3001, 2, 2)])
def test_attention_long_split(kv, batch, group):
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(kv)
    kv_lens = [kv - 7 * i for i in range(batch)]
    cache, table, ks, vs = filled(g, kv_lens, 64, 2, 128, spread=8.0)
    q = randn(g, batch, 2 * group, 128) * 2
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(starts([1] * batch)), return_lse=True, scale=0.2)
    check_attention(out, lse, q, ks, vs, kv_lens, starts([1] * batch), scale=0.2)


def test_attention_many_requests():
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(77)
    kv_lens = [(i * 37) % 90 for i in range(4096)]
    q_lens = [(i * 5) % 3 for i in range(4096)]
    cache, table, ks, vs = filled(g, kv_lens, 16, 1, 64)
    qs = starts(q_lens)
    q = randn(g, qs[-1], 2, 64)
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(qs), return_lse=True)
    check_attention(out, lse, q, ks, vs, kv_lens, qs)


def test_attention_extreme_sizes():
    """Scales far apart, queries near the ends of their type, large scores, zeros."""
    from vkccl_b200.ops.kv4 import kv4_attention, kv4_append, kv4_read

    g = gen(21)
    n = 200
    cache, table, _, _ = filled(g, [n], 16, 1, 128)
    kv = randn(g, n, 2, 128)
    kv[:, 1] *= (2.0 ** torch.randint(-12, 12, (n, 1), device="cuda", generator=g)).bfloat16()
    kv[50] = 0.0
    slots = (table[0].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16).int()
    kv4_append(cache, kv[:, :1], kv[:, 1:], slots)
    k, v = kv4_read(cache, slots, dtype=torch.float32)
    for f in (1.0, 2.0**-40, 2.0**40, 0.0):
        q = randn(g, 1, 8, 128) * f
        scale = 0.3 / f if f else 1.0
        out, lse = kv4_attention(q, cache, table, ints([n]), ints([0, 1]), return_lse=True, scale=scale)
        check_attention(out, lse, q, [k.double()], [v.double()], [n], [0, 1], scale=scale)


@pytest.mark.parametrize("scale", [-0.11, 0.0])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 3, 70]])
def test_attention_scale_is_any_number(scale, q_lens):
    """A negative scale turns the order of the scores, zero makes all weights equal; both kernels."""
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(23)
    kv_lens, qs = [700, 90, 333], starts(q_lens)
    cache, table, ks, vs = filled(g, kv_lens, 32, 1, 128)
    q = randn(g, qs[-1], 8, 128)
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(qs), return_lse=True, scale=scale)
    check_attention(out, lse, q, ks, vs, kv_lens, qs, scale=scale)


def test_attention_nan_where_it_belongs():
    """A NaN key or value reaches the rows that see it, and only those; garbage behind the end reaches none."""
    from vkccl_b200.ops.kv4 import kv4_attention, kv4_append

    g = gen(22)
    n, rows = 40, 10
    cache, table, ks, vs = filled(g, [n, n], 16, 1, 128)
    q = randn(g, 2 * rows, 8, 128)
    qs = starts([rows, rows])
    clean = kv4_attention(q, cache, table, ints([n, n]), ints(qs))
    kv = randn(g, 1, 2, 128)
    kv[0, 1, 100] = math.nan  # the value's second group of 64 channels
    slot = ints([int(table[0, 36 // 16]) * 16 + 36 % 16])
    kv4_append(cache, ks[0][36:37].bfloat16(), kv[:, 1:], slot)
    out = kv4_attention(q, cache, table, ints([n, n]), ints(qs))
    sees = torch.arange(rows, device="cuda") + n - rows + 1 > 36
    assert torch.isnan(out[:rows][sees][..., 64:]).all() and torch.isfinite(out[:rows][sees][..., :64]).all()
    assert torch.equal(out[:rows][~sees], clean[:rows][~sees]) and torch.equal(out[rows:], clean[rows:])
    kv[0, 0, 3] = math.inf
    kv4_append(cache, kv[:, :1], vs[0][36:37].bfloat16(), slot)
    out = kv4_attention(q, cache, table, ints([n, n]), ints(qs))
    assert torch.isnan(out[:rows][sees]).all() and torch.equal(out[:rows][~sees], clean[:rows][~sees])
    q[2, 3, 5] = math.nan
    out = kv4_attention(q, cache, table, ints([n, n]), ints(qs))
    assert torch.isnan(out[2, 3]).all() and torch.isfinite(out[2, 4]).all()


def test_attention_bad_pages_are_not_seen():
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(23)
    kv_lens = [100, 64]
    cache, table, ks, vs = filled(g, kv_lens, 16, 1, 128)
    q = randn(g, 2, 8, 128)
    bad = table.clone()
    bad[0, 1], bad[0, 4] = -1, cache.shape[0]
    bad[1, 0], bad[1, 3] = 2**31 - 1, -(2**31)
    out, lse = kv4_attention(q, cache, bad, ints(kv_lens), ints([0, 1, 2]), return_lse=True)
    keep0 = [i for i in range(100) if i // 16 not in (1, 4)]
    keep1 = [i for i in range(64) if i // 16 not in (0, 3)]
    check_attention(out, lse, q, [ks[0][keep0], ks[1][keep1]], [vs[0][keep0], vs[1][keep1]], [len(keep0), len(keep1)], [0, 1, 2])


def test_attention_corrupt_lengths_stay_in_bounds():
    """Lengths past the table and starts past the rows are cut; nothing outside of the tensors is touched."""
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(24)
    cache, table, ks, vs = filled(g, [32, 32], 16, 1, 64, width=2)
    q = randn(g, 2, 4, 64)
    out = kv4_attention(q, cache, table, ints([2**31 - 1, -5]), ints([0, 1, 2]))
    want = kv4_attention(q, cache, table, ints([32, 0]), ints([0, 1, 2]))
    assert torch.equal(out, want)
    out = kv4_attention(q, cache, table, ints([32, 32]), ints([0, 1, 2**31 - 1]))
    assert torch.equal(out, kv4_attention(q, cache, table, ints([32, 32]), ints([0, 1, 2])))
    kv4_attention(q, cache, table, ints([32, 32]), ints([7, -3, 1]))


def test_attention_out_strides_and_tail():
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(25)
    kv_lens, q_lens = [50, 70], [1, 3]
    cache, table, ks, vs = filled(g, kv_lens, 16, 2, 128)
    qkv = randn(g, 9, 12, 128)
    q = qkv[:, :8]
    want, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(starts(q_lens)), return_lse=True)
    out = torch.full((8, 9, 128), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    got = kv4_attention(q, cache, table, ints(kv_lens), ints(starts(q_lens)), out=out)
    assert got is out and torch.equal(out[:4], want[:4]) and (out[4:] == 7.0).all()
    assert (want[4:] == 0).all()
    assert kv4_attention(q[:0], cache, table, ints(kv_lens), ints([0, 0, 0])).shape == (0, 8, 128)


def test_attention_far_pages():
    """Pages behind 4 GiB of the cache."""
    from vkccl_b200.ops.kv4 import kv4_append, kv4_attention, kv4_read

    g = gen(26)
    pages, page, hk = 31000, 128, 8
    cache = torch.empty(pages, hk, page // 16, 18 * 128, dtype=torch.uint8, device="cuda")
    assert cache.numel() > 2**32
    n = 300
    table = ints([[pages - 1, pages - 2, 14563]])
    slots = (table[0].long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page).int()
    kv = randn(g, n, 2 * hk, 128)
    kv4_append(cache, kv[:, :hk], kv[:, hk:], slots)
    k, v = kv4_read(cache, slots, dtype=torch.float32)
    close(k, ref.stored_values(kv[:, :hk]), k.abs().double() * 2.0**-22, "far keys")
    q = randn(g, 1, 16, 128)
    out, lse = kv4_attention(q, cache, table, ints([n]), ints([0, 1]), return_lse=True)
    check_attention(out, lse, q, [k.double()], [v.double()], [n], [0, 1])


# ---- together, streams and graphs ---------------------------------------------------------


@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps_match_dense_attention(captured):
    """Prompts, then single tokens, with a request that ends and its row taken anew: every step's rows against
    dense attention in 64 bits over what was stored."""
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append_rope, kv4_attention
    from vkccl_b200.ops.paging import plan_pages

    g = gen(31)
    batch, page, width, hq, hk, dim, rows = 4, 16, 8, 8, 2, 128, 64
    pages = 20
    lens, count = torch.zeros(batch, dtype=torch.int32, device="cuda"), ints([pages])
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free, cache = ints(list(range(pages))), kv4_alloc(pages, page, hk, dim)
    new, finished = torch.zeros_like(lens), torch.zeros(batch, dtype=torch.bool, device="cuda")
    qkv = torch.zeros(rows, hq + 2 * hk, dim, dtype=torch.bfloat16, device="cuda")
    freq, w = inv_freq(dim), 1 + 0.1 * randn(g, dim)
    out = torch.zeros(rows, hq, dim, dtype=torch.bfloat16, device="cuda")
    lse = None
    held = {}

    def step():
        p = plan_pages(lens, new, table, free, count, page, rows, finished=finished, lens_out=lens, count_out=count)
        q = kv4_append_rope(cache, qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], p.slots, p.positions, freq,
                            q_weight=w, k_weight=w)
        kv4_attention(q, cache, table, p.kv_lens, p.q_starts, out=out)
        held["p"], held["q"] = p, q

    graph = None
    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()  # no rows yet
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    plans = [([30, 0, 17, 5], []), ([1, 40, 1, 1], []), ([1, 1, 1, 1], []), ([1, 1, 20, 1], [2]), ([1, 1, 1, 0], [3]),
             ([1, 1, 1, 33], [0])]
    history = [[] for _ in range(batch)]
    for n, ends in plans:
        qkv.copy_(randn(g, rows, hq + 2 * hk, dim))
        new.copy_(ints(n))
        finished.zero_()
        for i in ends:
            finished[i] = True
            history[i] = []
        graph.replay() if captured else step()
        qs = starts(n)
        ks, vs, kv_lens = [], [], []
        pos = held["p"].positions
        for i in range(batch):
            a, e = qs[i], qs[i + 1]
            assert pos[a:e].tolist() == list(range(len(history[i]), len(history[i]) + n[i]))
            rot = ref.norm_rope(qkv[a:e, hq:hq + hk], w, 1e-6, pos[a:e], freq, False)
            history[i] += list(zip(rot.bfloat16(), qkv[a:e, hq + hk:].clone()))
            kv_lens.append(len(history[i]))
            empty = torch.zeros(0, hk, dim, dtype=torch.float64, device="cuda")
            ks.append(ref.stored_values(torch.stack([h[0] for h in history[i]])) if history[i] else empty)
            vs.append(ref.stored_values(torch.stack([h[1] for h in history[i]])) if history[i] else empty)
        assert lens.tolist() == kv_lens
        q64 = ref.norm_rope(qkv[:, :hq], w, 1e-6, pos, freq, False)
        want = ref.attention(q64, ks, vs, kv_lens, qs, dim ** -0.5)[0]
        # bf16 queries and outputs, and keys whose 4-bit code may fall to the neighbour where the f32 and f64 rotations
        # round to neighbouring bf16 numbers: bounded in the norm of each row
        err = (out[:qs[-1]].double() - want[:qs[-1]]).norm(dim=-1) / (want[:qs[-1]].norm(dim=-1) + 1e-3)
        assert err.max().item() < 4 * 2.0**-8, err.max().item()


FIRST_CAPTURED = """
import torch
from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_attention
torch.manual_seed(1)
cache = kv4_alloc(8, 32, 1, 128)
k = torch.randn(256, 1, 128, device="cuda").bfloat16()
kv4_append(cache, k, k, torch.arange(256, device="cuda", dtype=torch.int32))
q = torch.randn(100, 8, 128, device="cuda").bfloat16()
table = torch.arange(8, device="cuda", dtype=torch.int32).view(1, 8)
lens, starts = torch.tensor([256], device="cuda", dtype=torch.int32), torch.tensor([0, 100], device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = kv4_attention(q, cache, table, lens, starts)
graph.replay()
want = kv4_attention(q, cache, table, lens, starts)
torch.cuda.synchronize()
assert got.abs().max() > 0 and torch.equal(got, want)
"""


def test_first_call_of_a_process_may_be_captured():
    """The word that reports a launch that gave up is made by the first call, inside the capture."""
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST_CAPTURED], capture_output=True, text=True, timeout=200)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_streams_and_shared_inputs():
    """Two attentions at once on two streams, over one cache, with scratch of their own."""
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(33)
    kv_lens = [2000, 900, 30]
    cache, table, _, _ = filled(g, kv_lens, 64, 2, 128)
    qa, qb = randn(g, 3, 16, 128), randn(g, 3, 16, 128)
    args = (cache, table, ints(kv_lens), ints([0, 1, 2, 3]))
    wa, wb = kv4_attention(qa, *args), kv4_attention(qb, *args)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(s1):
            a = kv4_attention(qa, *args)
        with torch.cuda.stream(s2):
            b = kv4_attention(qb, *args)
    torch.cuda.synchronize()
    assert torch.equal(a, wa) and torch.equal(b, wb)


def test_backward_captured_and_replayed():
    from vkccl_b200.ops.rope import qk_norm_rope_backward

    g = gen(34)
    q, k, w = randn(g, 100, 4, 64), randn(g, 100, 2, 64), 1 + 0.1 * randn(g, 64)
    dq, dk, pos, freq = randn(g, 100, 4, 64), randn(g, 100, 2, 64), ints(list(range(100))), inv_freq(64)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w)
    q.copy_(randn(g, 100, 4, 64))
    graph.replay()
    want = qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("qk_norm", [False, True])
def test_decode_model_with_cache(qk_norm):
    """TPLlamaDecode.step_cached on one rank: a prompt and two single tokens of two requests (one ends, its place is
    taken by a new prompt) against the same layers with attention in 64 bits over what was stored."""
    import vkccl_b200 as v
    from vkccl_b200.models.llama_decode import DecodeConfig, TPLlamaDecode
    from vkccl_b200.ops.fused import all_reduce_add_rms_norm
    from vkccl_b200.ops.gemm import gemm_bf16, gemm_silu_mul

    cfg = DecodeConfig(hidden=1024, intermediate=2048, heads=8, kv_heads=2, head_dim=128, layers=2, qk_norm=qk_norm,
                       page_size=16)
    comm = v.Communicator(1, v.get_unique_id(), 0, cuda_device=0)
    try:
        model, g = TPLlamaDecode(comm, cfg, seed=3), gen(40)
        cache = model.new_cache(2, 12, 96)
        stored = [[([], []) for _ in range(2)] for _ in range(cfg.layers)]  # layer, request -> keys, values
        held = [0, 0]
        for new, ends in (([37, 5], []), ([1, 1], []), ([1, 20], [1])):
            rows = sum(new) + 3
            x, xn = randn(g, rows, cfg.hidden), randn(g, rows, cfg.hidden)
            xr, xnr = x.clone(), xn.clone()
            done = torch.tensor([i in ends for i in range(2)], device="cuda")
            got = model.step_cached(x, xn, cache, ints(new), finished=done)
            qs = starts(new)
            for i in ends:
                held[i] = 0
                for layer in stored:
                    layer[i] = ([], [])
            pos = ints(sum(([held[i] + t for t in range(new[i])] for i in range(2)), []) + [0] * 3)
            held = [held[i] + new[i] for i in range(2)]
            for L, layer in zip(model.layers, stored):
                qkv = gemm_bf16(xnr, L["qkv"]).view(rows, 12, 128)
                q64 = ref.norm_rope(qkv[:, :8], L.get("qn"), cfg.eps, pos, model.inv_freq, False)
                k64 = ref.norm_rope(qkv[:, 8:10], L.get("kn"), cfg.eps, pos, model.inv_freq, False).bfloat16()
                ks, vs = [], []
                for i in range(2):
                    layer[i][0].append(ref.stored_values(k64[qs[i]:qs[i + 1]]))
                    layer[i][1].append(ref.stored_values(qkv[qs[i]:qs[i + 1], 10:]))
                    ks.append(torch.cat(layer[i][0]))
                    vs.append(torch.cat(layer[i][1]))
                attn = ref.attention(q64.bfloat16(), ks, vs, held, qs, 128 ** -0.5)[0].bfloat16()
                part = gemm_bf16(attn.view(rows, -1), L["o"])
                xnr = all_reduce_add_rms_norm(comm, part, xr, L["ln1"], cfg.eps)
                part = gemm_bf16(gemm_silu_mul(xnr, L["gu"]), L["d"])
                xnr = all_reduce_add_rms_norm(comm, part, xr, L["ln2"], cfg.eps)
            assert cache.lens.tolist() == held
            # The two differ where attention rounds to the neighbouring bf16 number (half a step, 2^-8, of its part of
            # the residual) and a 4-bit code to its neighbour; through two layers in the norm of a row.
            n = sum(new)
            err = (got[:n].double() - xnr[:n].double()).norm(dim=-1) / xnr[:n].double().norm(dim=-1)
            assert err.max().item() < 4 * 2.0**-8, err.max().item()
    finally:
        comm.destroy()
