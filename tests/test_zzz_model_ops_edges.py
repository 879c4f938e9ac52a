# SPDX-License-Identifier: Apache-2.0
"""The operators of a decode step over the 4-bit paged cache where they can go
wrong: sizes next to a limit, starts that no program should pass, values far
apart, scratch that is used again at once."""

import subprocess
import sys

import pytest
import torch

from conftest import ROOT, gpu_count

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if gpu_count() == 0:
        pytest.skip("no GPU")


# ---- plan ---------------------------------------------------------------------

PLAN_FIRST = """
import sys
import torch
from vkccl_b200.ops.paging import plan_pages
n = int(sys.argv[1])
i = lambda x: x.to(torch.int32)
ones = torch.ones(n, dtype=torch.int32, device="cuda")
table = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
free = i(torch.arange(n, device="cuda"))
p = plan_pages(torch.zeros_like(ones), ones, table, free, i(torch.tensor([n], device="cuda")), 16, n)
k = torch.arange(n, device="cuda")
assert torch.equal(table[:, 0], i(k)) and (table[:, 1] == -1).all() and torch.equal(p.slots, i(16 * k))
assert torch.equal(p.requests, i(k)) and torch.equal(p.q_starts, i(torch.arange(n + 1, device="cuda")))
assert (p.lens == 1).all() and (p.kv_lens == 1).all() and p.free_count.tolist() == [0]
"""


@pytest.mark.parametrize("batch", [6078, 6079, 6144, 6145])
def test_plan_first_of_a_process_takes_every_batch(batch):
    """Shared memory next to 48 KiB (8 bytes a request and the kernel's own 528): the limit is raised by the first call,
    whichever batch it has."""
    done = subprocess.run([sys.executable, "-c", PLAN_FIRST, str(batch)], capture_output=True, text=True, timeout=200, cwd=ROOT)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- attention: scratch ----------------------------------------------------------


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def raw_attention(q, cache, table, kv_lens, q_starts, out, workspace, zero_tail=0):
    """The library's entry with scratch of the caller's."""
    from vkccl_b200._lib import lib
    from vkccl_b200.ops import _args

    dev, (t, n, dim), (batch, width) = q.get_device(), q.shape, table.shape
    c, _, _, _ = _args.cache4(cache, dim, dev)
    _args.call(lib().vcclKv4Attention, "vcclKv4Attention", dev, _args.heads(q, "q", q.dtype, dev, t, dim), c, table.data_ptr(), width,
               kv_lens.data_ptr(), q_starts.data_ptr(), batch, t, dim ** -0.5, _args.heads(out, "out", q.dtype, dev, t, dim, n, True),
               None, zero_tail, workspace.data_ptr(), _args.DTYPES[q.dtype])


def workspace_bytes(batch, tokens, heads, kv_heads, dim):
    from vkccl_b200._lib import lib

    return lib().vcclKv4AttentionWorkspace(batch, tokens, heads, kv_heads, dim)


def random_cache(g, pages, page, kv_heads, dim):
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append

    cache = kv4_alloc(pages, page, kv_heads, dim)
    kv = torch.randn(pages * page, 2 * kv_heads, dim, device="cuda", generator=g).bfloat16()
    kv4_append(cache, kv[:, :kv_heads], kv[:, kv_heads:], torch.arange(pages * page, dtype=torch.int32, device="cuda"))
    return cache


@pytest.mark.parametrize("tokens,starts", [(4096, [0, 1000, 2000, 3000, 4096]), (640, [0, 0, 0, 0, 0])])
def test_scratch_is_free_when_the_call_is_over(tokens, starts):
    """Requests that are all long, or no rows at all: the next kernel on the stream may take the scratch, whichever of the
    call's kernels had anything to do."""
    g = gen(1)
    cache, table = random_cache(g, 16, 64, 8, 128), torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4)
    q = torch.randn(tokens, 64, 128, device="cuda", generator=g).bfloat16()
    kv, qs = ints([256] * 4), ints(starts)
    out = torch.zeros_like(q)
    size = workspace_bytes(4, tokens, 64, 8, 128)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    raw_attention(q, cache, table, kv, qs, out, ws)
    want = out.clone()
    touched = torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(100):
        raw_attention(q, cache, table, kv, qs, out, ws)
        ws.fill_(0xA5)
        touched |= (ws != 0xA5).any()
    assert not touched.item() and torch.equal(out, want)


@pytest.mark.parametrize("tokens,heads,kv_heads,starts", [(100, 8, 1, [0, 100, 0, 100, 0]), (100, 8, 1, [100, 0, 100, 0, 100] * 8),
                                                          (3000, 64, 8, [0, 3000, 0, 3000, -5, 3000, 7]), (100, 8, 1, [0, 30, 100])])
def test_attention_starts_that_fall_stay_in_bounds(tokens, heads, kv_heads, starts):
    """Rows that several requests claim make more work than the scratch was sized for: what has no room is left out."""
    g = gen(2)
    batch = len(starts) - 1
    cache = random_cache(g, 20, 16, kv_heads, 128)
    table = torch.arange(20, dtype=torch.int32, device="cuda").repeat(batch, 1)
    q = torch.randn(tokens, heads, 128, device="cuda", generator=g).bfloat16()
    size = workspace_bytes(batch, tokens, heads, kv_heads, 128)
    ws = torch.full((size + (4 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    rows = torch.full((tokens + 64, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    raw_attention(q, cache, table, ints([320 - i for i in range(batch)]), ints(starts), rows[:tokens], ws)
    assert (ws[size:] == 0xA5).all() and (rows[tokens:] == 7.0).all()


# ---- attention: values and keys far apart ----------------------------------------


def spread_case(g, kind, n, kv_heads, ratio, dim=128):
    """Keys and values [n, kv heads, 128] for queries around 0.5: a key of a * ones has a score of 5.7 a (4 a with 64 channels)."""
    def noise(x):
        return x * torch.randn(n, kv_heads, dim, device="cuda", generator=g)

    t = torch.arange(n, device="cuda", dtype=torch.float64)[:, None, None] / n
    k, v = noise(0.2), noise(1.0)
    if kind in ("first", "middle", "last"):  # one value is large, and its weight is nothing
        i = {"first": 0, "middle": n // 2 + 5, "last": n - 1}[kind]
        v[i] *= 2.0**ratio
        k[i] = k[i] - 40.0
    elif kind == "unseen":  # the last token's value is large: its own row sees it alone
        v[n - 1] *= 2.0**ratio
    elif kind == "sink":  # the first token has most of the weight and small values
        v[0] *= 2.0**-ratio
        k[0] = k[0] + 1.0
    elif kind == "rising":  # what comes later counts more and is smaller
        v, k = v * 2.0**(-ratio * t), k + 12.0 * t
    elif kind == "falling":  # what comes later counts less and is larger: by less than it counts less ...
        v, k = v * 2.0**(ratio * t), k - 12.0 * t
    elif kind == "growing":  # ... and by more
        v, k = v * 2.0**(ratio * t), k - 2.0 * t
    elif kind == "groups":  # some tokens' first 64 channels far above their others, which are like the rest
        v[..., :64] *= torch.where(torch.rand(n, kv_heads, 1, device="cuda", generator=g) < 0.05, 2.0**ratio, 1.0)
    elif kind == "key unseen":
        k[n - 1] *= 2.0**ratio
    elif kind == "key below":  # one key is large, and its weight is nothing
        k[n // 2 + 5] = k[n // 2 + 5] - 2.0**ratio
    elif kind == "mixed":  # neighbours far apart
        v = v * 2.0**torch.randint(-ratio, ratio + 1, (n, kv_heads, 1), device="cuda", generator=g)
    return k, v


def check_rows(got, lse, q, ks, vs, kv_lens, q_starts, long):
    """Each row against 64 bits, within a slack from the values that it sees itself.

    With a the largest |value| of a token's 64 channels and A = sum p a over the row: the weights are rounded to f16, 2^-11
    of 7.5 scales <= 1.01 a; in the kernel of long runs the value too, twice (2.1 * 2^-11 a).  What falls under f16's
    smallest numbers is 2^-27 A a token for single tokens (weights in units of the largest p * scale seen, times 4), and 2^-20 A
    in long runs (where 32 tokens within 2^6 share their unit).  f32 sums of n terms and exponentials: 2^-15.  Scores are
    off by 2^-19 of the sizes that they add up."""
    import model_reference as ref

    scale = q.shape[-1] ** -0.5
    want, wlse, _ = ref.attention(q, ks, vs, kv_lens, q_starts, scale)
    tops = [v.abs().unflatten(-1, (-1, 64)).amax(-1, keepdim=True).expand(*v.shape[:-1], -1, 64).flatten(-2) for v in vs]
    _, _, size = ref.attention(q, ks, tops, kv_lens, q_starts, scale)
    # sum |q| |k| of a row against the keys of weight: those are near the row's largest score
    _, _, near = ref.attention(q, ks, [k.abs().amax(-1, keepdim=True).expand_as(k) * 2 for k in ks], kv_lens, q_starts, scale)
    score = q.double().abs().sum(-1) * near[..., 0] * scale * 2.0**-19
    n = max(kv_lens)
    part = (3.2 * 2.0**-11 + n * 2.0**-20 if long else 1.1 * 2.0**-11 + n * 2.0**-27) + 2.0**-15
    slack = want.abs() * torch.finfo(q.dtype).eps / 2 * 1.02 + size * (part + 4 * score[..., None]) + 2.0**-25
    d = (got.double() - want).abs() - slack
    assert torch.isfinite(got).all() and d.max().item() <= 0, (d.max().item(), (d / slack).max().item())
    assert ((lse.double() - wlse).abs() <= score + wlse.abs() * 2.0**-20 + 2.0**-18).all()


KINDS = ["first", "middle", "last", "unseen", "sink", "rising", "falling", "growing", "mixed", "key unseen", "key below", "groups"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ratio", [14, 26])
@pytest.mark.parametrize("rows,heads,kv_heads,n,dim", [(1, 8, 1, 2000, 128), (3, 2, 1, 700, 128), (40, 2, 2, 700, 64), (100, 8, 1, 700, 128),
                                                       (100, 4, 2, 690, 64), (1100, 64, 8, 1100, 128)])
def test_attention_of_values_far_apart(kind, ratio, rows, heads, kv_heads, n, dim):
    """Values (and keys) of one request 2^14 and 2^26 apart: a row's result goes by the tokens that it sees and by their weights,
    not by the largest value around.  One row, a few, and runs of rows with and without shares of the keys."""
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_attention, kv4_read

    long = rows * heads // kv_heads >= 64
    if kind == "groups" and long and ratio > 14:
        ratio = 14  # the groups of a row share its weights there: bits of the smaller one's go from 2^16 on
    g = gen(KINDS.index(kind) * 100 + ratio + rows)
    pages = -(-n // 16)
    cache = kv4_alloc(pages, 16, kv_heads, dim)
    table = torch.randperm(pages, device="cuda", generator=g).int().view(1, -1)
    t = torch.arange(n, device="cuda")
    slots = (table[0, t // 16] * 16 + t % 16).int()
    k, v = spread_case(g, kind, n, kv_heads, ratio, dim)
    kv4_append(cache, k.bfloat16(), v.bfloat16(), slots)
    k, v = (x.double() for x in kv4_read(cache, slots, dtype=torch.float32))
    q = (0.5 + 0.1 * torch.randn(rows, heads, dim, device="cuda", generator=g)).bfloat16()
    got, lse = kv4_attention(q, cache, table, ints([n]), ints([0, rows]), return_lse=True)
    check_rows(got, lse, q, [k], [v], [n], [0, rows], long)


def test_attention_of_a_long_run_among_the_largest_batch():
    """4096 requests, one of them with 300 rows: the starts of all of them stand in shared memory beside the tiles."""
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(5)
    q_lens, kv_lens = [1] * 4096, [1 + i % 16 for i in range(4096)]
    q_lens[1234], kv_lens[1234] = 300, 320
    cache = random_cache(g, 60, 16, 1, 128)
    table = torch.randint(0, 60, (4096, 20), device="cuda", generator=g).int()
    qs = [0] + torch.tensor(q_lens).cumsum(0).tolist()
    q = torch.randn(qs[-1], 32, 128, device="cuda", generator=g).bfloat16()  # 32 query heads on one: 24 rows a request and more
    got, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(qs), return_lse=True)
    some = [0, 1, 1233, 1234, 1235, 4095]
    rows = torch.cat([torch.arange(qs[i], qs[i + 1], device="cuda") for i in some])
    one, lse1 = kv4_attention(q[rows], cache, table[some], ints([kv_lens[i] for i in some]),
                              ints([0] + torch.tensor([q_lens[i] for i in some]).cumsum(0).tolist()), return_lse=True)
    # the same rows among few requests: shares of the keys differ, and with them f32 sums and one rounding of each weight
    assert (got[rows].float() - one.float()).abs().max() <= 2.0**-6 and (lse[rows] - lse1).abs().max() <= 2.0**-16
    assert torch.isfinite(got).all()


# ---- a launch that gave up ---------------------------------------------------------


def test_attention_that_gave_up_is_reported():
    """The word that a launch whose wait ran out leaves behind (set from the host): the next call raises and the one after
    works; replays of a captured call raise nothing, and the look after them does, once."""
    import vkccl_b200 as v
    from vkccl_b200._lib import lib
    from vkccl_b200.ops.kv4 import kv4_attention, kv4_attention_status

    g = gen(6)
    cache, table = random_cache(g, 16, 16, 1, 128), torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    q = torch.randn(100, 8, 128, device="cuda", generator=g).bfloat16()
    args = (cache, table, ints([256]), ints([0, 100]))
    want = kv4_attention(q, *args)
    kv4_attention_status()
    assert lib().vcclxKv4AttentionInjectAbort() == 0
    with pytest.raises(v.VcclError):
        kv4_attention(q, *args)
    assert torch.equal(kv4_attention(q, *args), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv4_attention(q, *args)
    assert lib().vcclxKv4AttentionInjectAbort() == 0
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(v.VcclError):
        kv4_attention_status("cuda:0")
    kv4_attention_status()
    assert torch.equal(got, want) and torch.equal(kv4_attention(q, *args), want)


# ---- the decode step ---------------------------------------------------------------


def test_decode_step_tells_which_requests_were_refused():
    """Three requests and pages for two prompts: the third's rows come back, and the plan says that they saw nothing."""
    import vkccl_b200 as v
    from vkccl_b200.models.llama_decode import DecodeConfig, TPLlamaDecode

    cfg = DecodeConfig(hidden=1024, intermediate=2048, heads=8, kv_heads=2, head_dim=128, layers=1, page_size=16)
    comm = v.Communicator(1, v.get_unique_id(), 0, cuda_device=0)
    try:
        model, g = TPLlamaDecode(comm, cfg, seed=3), gen(7)
        x = torch.randn(60, 1024, device="cuda", generator=g).bfloat16()
        plain = model.step_cached(x.clone(), x, model.new_cache(3, 4, 64), ints([20, 20, 20]))
        cache = model.new_cache(3, 4, 64)
        got, plan = model.step_cached(x.clone(), x, cache, ints([20, 20, 20]), return_plan=True)
        assert torch.equal(got, plain)
        assert plan.kv_lens.tolist() == [20, 20, 0] and cache.lens.tolist() == [20, 20, 0]
        assert (plan.slots[40:] == -1).all() and (plan.slots[:40] >= 0).all()
        assert cache.free_count.tolist() == plan.free_count.tolist() == [0]
    finally:
        comm.destroy()


# ---- gradients ---------------------------------------------------------------------


def test_norm_rope_inside_an_autograd_function():
    """The way to train with it: the forward call runs without grad mode, the backward call is explicit."""
    import model_reference as ref
    from vkccl_b200.ops.rope import qk_norm_rope, qk_norm_rope_backward

    class NormRope(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, pos, freq, w):
            ctx.save_for_backward(q, k, pos, freq, w)
            return qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w)

        @staticmethod
        def backward(ctx, dq, dk):
            q, k, pos, freq, w = ctx.saved_tensors
            dq, dk, a, b = qk_norm_rope_backward(dq.contiguous(), dk.contiguous(), q, k, pos, freq, q_weight=w, k_weight=w)
            return dq, dk, None, None, a + b

    g = gen(8)
    q, k = (torch.randn(37, n, 64, device="cuda", generator=g).bfloat16().requires_grad_() for n in (4, 2))
    w = (1 + 0.1 * torch.randn(64, device="cuda", generator=g)).bfloat16().requires_grad_()
    pos, freq = torch.arange(37, dtype=torch.int32, device="cuda"), (100.0 ** (-torch.arange(32, device="cuda") / 32)).float()
    dq, dk = (torch.randn(37, n, 64, device="cuda", generator=g).bfloat16() for n in (4, 2))
    with pytest.raises(ValueError):
        qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w)
    yq, yk = NormRope.apply(q, k, pos, freq, w)
    torch.autograd.backward([yq, yk], [dq, dk])
    q64, k64, w64 = (x.detach().double().requires_grad_() for x in (q, k, w))
    ((ref.norm_rope(q64, w64, 1e-6, pos, freq, False) * dq.double()).sum()
     + (ref.norm_rope(k64, w64, 1e-6, pos, freq, False) * dk.double()).sum()).backward()
    for x, y in ((q, q64), (k, k64)):
        # half a step of bf16 and f32 arithmetic on terms up to a few times the largest gradient of the row
        slack = y.grad.abs() * 2.0**-8 * 1.02 + 2.0**-16 * y.grad.abs().amax(-1, keepdim=True)
        assert ((x.grad.double() - y.grad).abs() <= slack).all()
    # two sums rounded to bf16, added and rounded: each half a step of its size (at most the sum of the terms' sizes)
    assert ((w.grad.double() - w64.grad).abs() <= 3 * 2.0**-8 * (w64.grad.abs() + 30)).all()


# ---- long runs of rows: what the short ones are tested for -------------------------


@pytest.mark.parametrize("q_lens,kv_lens", [([300, 7, 100], [0, 3, 40]), ([90] * 40, [0, 1, 89, 90, 91, 63, 64, 65, 127, 200] * 4)])
@pytest.mark.parametrize("page", [16, 48])
def test_long_runs_without_keys_and_with_fewer_keys_than_rows(q_lens, kv_lens, page):
    """Requests of many rows that hold nothing, or fewer tokens than rows, with and without shares of the keys; pages of 48."""
    from test_zzz_kv4 import check_attention, filled, starts
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(11)
    cache, table, ks, vs = filled(g, kv_lens, page, 8, 128)
    qs = starts(q_lens)
    q = torch.randn(qs[-1] + 5, 16, 128, device="cuda", generator=g).bfloat16()
    out, lse = kv4_attention(q, cache, table, ints(kv_lens), ints(qs), return_lse=True)
    check_attention(out, lse, q, ks, vs, kv_lens, qs)
    assert out[qs[-1]:].abs().max() == 0 and torch.isinf(lse[qs[-1]:]).all()
    again = kv4_attention(q, cache, table, ints(kv_lens), ints(qs))
    assert torch.equal(out, again)


def test_long_runs_do_not_see_bad_pages():
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(12)
    n, rows = 300, 40
    cache = random_cache(g, 40, 16, 1, 128)
    table = torch.randperm(40, device="cuda", generator=g).int()[:19].view(1, 19)
    bad = table.clone()
    bad[0, 3], bad[0, 7], bad[0, 8] = -1, cache.shape[0], 2**31 - 1
    q = torch.randn(rows, 8, 128, device="cuda", generator=g).bfloat16()
    out, lse = kv4_attention(q, cache, bad, ints([n]), ints([0, rows]), return_lse=True)
    keep = [i for i in range(19) if i not in (3, 7, 8)]
    # the pages that are left, in order: the last rows see the same tokens, 48 fewer
    want, wlse = kv4_attention(q, cache, table[:, keep].contiguous(), ints([n - 48]), ints([0, rows]), return_lse=True)
    # sums of the same terms in other tiles: f32, and weights rounded to f16 in other units
    assert (out.float() - want.float()).abs().max() <= 2.0**-7 and (lse - wlse).abs().max() <= 2.0**-16


@pytest.mark.parametrize("dtype,f", [(torch.bfloat16, 2.0**-60), (torch.bfloat16, 2.0**60), (torch.bfloat16, 2.0**-112),
                                     (torch.bfloat16, 2.0**124), (torch.bfloat16, 0.0), (torch.float16, 2.0**-13),
                                     (torch.float16, 2.0**12)])
@pytest.mark.parametrize("rows", [2, 30])
def test_queries_of_every_size(dtype, f, rows):
    """Queries next to the ends of their type, the scale making up for it: few rows and long runs."""
    from test_zzz_kv4 import check_attention, filled
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(13)
    cache, table, ks, vs = filled(g, [500], 16, 2, 128)
    q = (torch.randn(rows, 16, 128, device="cuda", generator=g) * f).to(dtype)
    scale = 0.1 / f if f else 0.1
    out, lse = kv4_attention(q, cache, table, ints([500]), ints([0, rows]), return_lse=True, scale=scale)
    check_attention(out, lse, q, ks, vs, [500], [0, rows], scale=scale)


@pytest.mark.parametrize("dim,rot", [(24, 16), (40, 32), (72, 64), (104, 48), (136, 128), (200, 112), (248, 240)])
@pytest.mark.parametrize("inter", [False, True])
def test_norm_rope_of_odd_head_dimensions(dim, rot, inter):
    """Head dimensions that are multiples of 8 and not of 16: a row's halves end inside of 8 channels."""
    import model_reference as ref
    from test_zzz_kv4 import close, inv_freq, rope_slack
    from vkccl_b200.ops.rope import qk_norm_rope, qk_norm_rope_backward

    g = gen(dim)
    tokens, w = 53, (1 + 0.2 * torch.randn(dim, device="cuda", generator=g)).bfloat16()
    q, k, dq, dk = (torch.randn(tokens, n, dim, device="cuda", generator=g).bfloat16() for n in (3, 1, 3, 1))
    pos, freq = ints([i * 1001 for i in range(tokens)]), inv_freq(rot)
    out = torch.full((tokens, 5, dim), 7.0, device="cuda").bfloat16()
    yq, yk = qk_norm_rope(q, k, pos, freq, q_weight=w, k_weight=w, interleaved=inter, q_out=out[:, :3], k_out=out[:, 3:4])
    assert (out[:, 4] == 7.0).all()
    gq, gk, dwq, dwk = qk_norm_rope_backward(dq, dk, q, k, pos, freq, q_weight=w, k_weight=w, interleaved=inter)
    for x, y, d, dx, dw in ((q, yq, dq, gq, dwq), (k, yk, dk, gk, dwk)):
        leaf, wl = x.double().requires_grad_(), w.double().requires_grad_()
        want = ref.norm_rope(leaf, wl, 1e-6, pos, freq, inter)
        close(y, want.detach(), rope_slack(want.detach(), torch.bfloat16, want.detach().abs().amax(-1, keepdim=True)), "forward")
        (want * d.double()).sum().backward()
        size = leaf.grad.abs().amax(-1, keepdim=True) + d.double().abs().amax(-1, keepdim=True) * 6 / x.double().square().mean(-1, keepdim=True).sqrt()
        close(dx, leaf.grad, rope_slack(leaf.grad, torch.bfloat16, size), "dx")
        # terms |g x^| of at most 6 * 6, f32 sums of a lane's rows
        close(dw, wl.grad, wl.grad.abs() * 2.0**-8 + tokens * 3 * 36 * 2.0**-20, "dw")


# ---- attention: long sums ----------------------------------------------------------


@pytest.mark.parametrize("rows,heads", [(1, 64), (2, 8), (16, 64)])
def test_attention_of_many_long_contexts(rows, heads):
    """250 requests of 60000 tokens (of the same pages): a warp adds up whole requests, and the error must not grow with them.

    In the norm of a row: the output is rounded to f16 (2^-11 of it at most), and every weight (2^-11 of p * 7.5 scales <= 1.01 p a, a
    the largest |value| of the token's 64 channels, which add up as sqrt(sum p^2 a^2): the roundings of different tokens have
    nothing to do with one another).  The tensor cores add 16 tokens a step to an f32 and drop what is below its last bit, 2^-23 of
    it at most: n / 16 steps of the row itself, and for single tokens 8 steps of what 128 tokens add up to before the middle of
    their codes is taken out, codes up to 255 / 16 of a scale where values go to 7.5 of it (2.2 a, half of it on average).  Runs of
    rows round every value twice (2.1 * 2^-11 a)."""
    from vkccl_b200.ops.kv4 import kv4_attention, kv4_read

    g = gen(14)
    n, batch, page, kv_heads = 60000, 250, 64, 8
    pages = -(-n // page)
    cache = random_cache(g, pages, page, kv_heads, 128)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)
    q = (torch.randn(batch * rows, heads, 128, device="cuda", generator=g) * 0.5).half()
    out = kv4_attention(q, cache, table, ints([n] * batch), ints([i * rows for i in range(batch + 1)]))
    k, v = (x.double() for x in kv4_read(cache, torch.arange(n, dtype=torch.int32, device="cuda"), dtype=torch.float32))
    tops = v.abs().unflatten(-1, (-1, 64)).amax(-1)  # [n, kv heads, 2]
    for t in (0, 7 * rows, 249 * rows):
        for h in (0, heads - 1):
            j = h // (heads // kv_heads)
            see = n - (rows - 1 - t % rows)
            p = torch.softmax(k[:see, j] @ q[t, h].double() * 128 ** -0.5, 0)
            want = p @ v[:see, j]
            a = tops[:see, j].repeat_interleave(64, -1)
            roundings = 3.1 if rows * heads // kv_heads >= 64 else 1.01
            slack = ((want.norm() + (p.square() @ a.square()).sqrt().norm() * roundings) * 2.0**-11 + want.norm() * n / 16 * 2.0**-23
                     + (p @ a).norm() * 8 * 1.1 * 2.0**-23)
            d = (out[t, h].double() - want).norm()
            assert d <= slack, (t, h, d.item(), slack.item(), want.norm().item())


# ---- calls at once -------------------------------------------------------------------


def test_long_runs_on_two_streams_beside_a_gemm():
    """Kernels that take all of an SM's tensor memory, beside one that takes a part of it: the same bits as one after another."""
    from vkccl_b200.ops.gemm import gemm_bf16
    from vkccl_b200.ops.kv4 import kv4_attention

    g = gen(15)
    cache, table = random_cache(g, 64, 16, 2, 128), torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32)
    args = (cache, table, ints([500, 512]), ints([0, 200, 300]))
    qa, qb = (torch.randn(300, 16, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
    x, w = (torch.randn(n, 1024, device="cuda", generator=g).bfloat16() for n in (512, 2048))
    want = kv4_attention(qa, *args), kv4_attention(qb, *args), gemm_bf16(x, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, f in zip(streams, (lambda: kv4_attention(qa, *args), lambda: kv4_attention(qb, *args), lambda: gemm_bf16(x, w))):
            with torch.cuda.stream(s):
                got.append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))


def test_constant_values_and_a_late_scale():
    """Groups of equal channels have a scale of zero, and no weight of f16 goes by it; behind them come ordinary ones."""
    from test_zzz_kv4 import check_attention
    from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append, kv4_attention, kv4_read

    g = gen(16)
    n = 400
    cache, table = kv4_alloc(25, 16, 1, 128), torch.arange(25, dtype=torch.int32, device="cuda").view(1, 25)
    kv = torch.randn(n, 2, 128, device="cuda", generator=g).bfloat16()
    kv[:300, 1] = kv[:300, 1, :1]  # all channels of a token's value alike
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    kv4_append(cache, kv[:, :1], kv[:, 1:], slots)
    k, v = (x.double() for x in kv4_read(cache, slots, dtype=torch.float32))
    for rows in (1, 3, 120):
        for length in (299, 301, n):
            q = torch.randn(rows, 8, 128, device="cuda", generator=g).bfloat16()
            out, lse = kv4_attention(q, cache, table, ints([length]), ints([0, rows]), return_lse=True)
            check_attention(out, lse, q, [k[:length]], [v[:length]], [length], [0, rows])
