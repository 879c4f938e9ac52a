# SPDX-License-Identifier: Apache-2.0
"""Refusals of the model operators (page plan, norm + rotation, 4-bit cache),
without a GPU: the C entries return vcclInvalidArgument before they launch
anything, and the Python checks raise ValueError."""

import ctypes
import struct

import pytest
import torch

from vkccl_b200._lib import lib
from vkccl_b200.ops import _args
from vkccl_b200.ops import kv4, paging, rope

OK, INVALID = 0, 4
BF16, F16, F32, I32 = 9, 6, 7, 2
CPU = -1  # the device number of a CPU tensor


def heads(at=4096, tok=512, head=128, n=4):
    return struct.pack("@Pqqi4x", at, tok, head, n)


def rope_c(pos=4096, freq=4096, wq=0, wk=0, half=64, inter=0, eps=1e-6):
    return struct.pack("@PPPPiif4x", pos, freq, wq, wk, half, inter, eps)


def cache_c(at=4096, pages=2, page=16, n=4, dim=128):
    return struct.pack("@Piiii", at, pages, page, n, dim)


P = 4096  # an address that a refused call never follows


def test_structure_sizes():
    class H(ctypes.Structure):
        _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_longlong), ("c", ctypes.c_longlong), ("d", ctypes.c_int)]

    class R(ctypes.Structure):
        _fields_ = [(x, ctypes.c_void_p) for x in "abcd"] + [("e", ctypes.c_int), ("f", ctypes.c_int), ("g", ctypes.c_float)]

    class K(ctypes.Structure):
        _fields_ = [("a", ctypes.c_void_p)] + [(x, ctypes.c_int) for x in "bcde"]

    assert (len(heads()), len(rope_c()), len(cache_c())) == (ctypes.sizeof(H), ctypes.sizeof(R), ctypes.sizeof(K))


def plan(**kw):
    d = dict(lens=P, new=P, fin=None, table=P, free=P, count=P, batch=4, width=4, pool=8, page=16, tokens=4, pos=P, slots=P,
             req=P, qs=P, kv=P, lo=P, co=P, fp=P, stream=None)
    d.update(kw)
    return lib().vcclPagePlan(*d.values())


@pytest.mark.parametrize("bad", [dict(lens=None), dict(new=None), dict(table=None), dict(free=None), dict(count=None), dict(qs=None),
                                 dict(kv=None), dict(lo=None), dict(co=None), dict(fp=None), dict(batch=0), dict(batch=8193),
                                 dict(width=0), dict(pool=0), dict(page=0), dict(tokens=-1), dict(pos=None), dict(slots=None),
                                 dict(req=None), dict(pool=1 << 28, page=16), dict(width=1 << 28, page=16)])
def test_plan_refuses(bad):
    assert plan(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(q=heads(at=0)), dict(q=heads(at=P + 8)), dict(q=heads(tok=514)), dict(k=heads(head=4)),
                                 dict(k=heads(n=0)), dict(k=heads(n=40000)), dict(q=heads(tok=1 << 31)), dict(q=heads(tok=-512)),
                                 dict(qo=heads(n=5)), dict(ko=heads(n=3)), dict(ko=heads(at=0)), dict(tokens=-1), dict(dim=0),
                                 dict(dim=124), dict(dim=264), dict(dt=F32), dict(dt=I32), dict(r=rope_c(half=4)),
                                 dict(r=rope_c(half=60)), dict(r=rope_c(half=72)), dict(r=rope_c(half=0)), dict(r=rope_c(eps=-1.0)),
                                 dict(r=rope_c(eps=float("nan"))), dict(r=rope_c(pos=0)), dict(r=rope_c(freq=0)), dict(r=None),
                                 dict(r=rope_c(wq=P + 2)), dict(q=None)])
def test_norm_rope_refuses(bad):
    d = dict(q=heads(), k=heads(), r=rope_c(), qo=heads(), ko=heads(), tokens=3, dim=128, dt=BF16, stream=None)
    d.update(bad)
    assert lib().vcclQkNormRope(*d.values()) == INVALID


def test_norm_rope_of_no_tokens_is_nothing():
    assert lib().vcclQkNormRope(None, None, rope_c(), None, None, 0, 128, BF16, None) == OK


@pytest.mark.parametrize("bad", [dict(dq=heads(n=3)), dict(q=heads(at=0)), dict(dqi=heads(n=2)), dict(wq=None), dict(wk=None), dict(ws=None),
                                 dict(r=rope_c()), dict(r=rope_c(wq=P)), dict(dim=300), dict(dt=F32)])
def test_backward_refuses(bad):
    d = dict(dq=heads(), dk=heads(), q=heads(), k=heads(), r=rope_c(wq=P, wk=P), dqi=heads(), dki=heads(), wq=P, wk=P, ws=P, tokens=3,
             dim=128, dt=BF16, stream=None)
    d.update(bad)
    assert lib().vcclQkNormRopeBackward(*d.values()) == INVALID


BAD_CACHES = [cache_c(at=0), cache_c(at=P + 4), cache_c(pages=0), cache_c(page=0), cache_c(page=24), cache_c(n=0), cache_c(dim=96),
              cache_c(pages=1 << 28, page=16), None]


@pytest.mark.parametrize("bad", [dict(c=c) for c in BAD_CACHES] +
                         [dict(k=heads(n=3)), dict(v=heads(n=5)), dict(slots=None), dict(tokens=-1), dict(dt=F32), dict(k=None),
                          dict(r=rope_c()), dict(r=rope_c(), q=heads()), dict(q=heads(), qo=heads()),
                          dict(r=rope_c(), q=heads(), qo=heads(n=3)), dict(r=rope_c(half=4), q=heads(), qo=heads())])
def test_append_refuses(bad):
    d = dict(c=cache_c(), k=heads(), v=heads(), slots=P, r=None, q=None, qo=None, tokens=2, dt=BF16, stream=None)
    d.update(bad)
    assert lib().vcclKv4Append(*d.values()) == INVALID


@pytest.mark.parametrize("bad", [dict(c=c) for c in BAD_CACHES] + [dict(slots=None), dict(k=heads(n=1)), dict(v=heads(head=14)), dict(dt=I32)])
def test_read_refuses(bad):
    d = dict(c=cache_c(), slots=P, k=heads(), v=heads(), tokens=2, dt=F32, stream=None)
    d.update(bad)
    assert lib().vcclKv4Read(*d.values()) == INVALID


@pytest.mark.parametrize("bad", [dict(c=c) for c in BAD_CACHES] +
                         [dict(q=heads(n=6)), dict(o=heads(n=8)), dict(o=None), dict(table=None), dict(width=0), dict(kv=None),
                          dict(qs=None), dict(batch=0), dict(batch=4097), dict(tokens=-1), dict(ws=None), dict(dt=F32),
                          dict(width=1 << 28), dict(q=heads(n=30000), o=heads(n=30000), tokens=1 << 20)])
def test_attention_refuses(bad):
    d = dict(q=heads(n=4), c=cache_c(), table=P, width=2, kv=P, qs=P, batch=2, tokens=2, scale=0.1, o=heads(n=4), lse=None, zero=1, ws=P,
             dt=BF16, stream=None)
    d.update(bad)
    assert lib().vcclKv4Attention(*d.values()) == INVALID


def test_workspaces_are_sized_without_a_gpu():
    h = lib()
    assert h.vcclQkNormRopeBackwardWorkspace(128) > 0 and h.vcclQkNormRopeBackwardWorkspace(0) == 0
    small, large = (h.vcclKv4AttentionWorkspace(4, t, 8, 1, 128) for t in (4, 4000))
    assert 0 < small < large
    for bad in ((0, 4, 8, 1, 128), (4, -1, 8, 1, 128), (4, 4, 0, 1, 128), (4, 4, 8, 0, 128), (4, 4, 1, 8, 128), (4, 4, 8, 1, 0)):
        assert h.vcclKv4AttentionWorkspace(*bad) == 0


# ---- Python checks ---------------------------------------------------------------


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        paging.plan_pages(i, i, torch.zeros(4, 2, dtype=torch.int32), i, i[:1], 16, 4)
    with pytest.raises(ValueError):
        rope.qk_norm_rope(t(4, 2, 64), t(4, 2, 64), i, torch.zeros(32))
    with pytest.raises(ValueError):
        kv4.kv4_append(t(2, 1, 1, 1152, dtype=torch.uint8), t(4, 1, 64), t(4, 1, 64), i)
    with pytest.raises(ValueError):
        kv4.kv4_read(t(2, 1, 1, 1152, dtype=torch.uint8), i)
    with pytest.raises(ValueError):
        kv4.kv4_attention(t(4, 1, 64), t(2, 1, 1, 1152, dtype=torch.uint8), i.view(1, 4), i[:1], i[:2])


@pytest.mark.parametrize("args", [(4, 16, 1, 96), (4, 24, 1, 64), (4, 0, 1, 64), (0, 16, 1, 64), (4, 16, 0, 64), (1 << 28, 16, 1, 64)])
def test_alloc_refuses(args):
    with pytest.raises(ValueError):
        kv4.kv4_alloc(*args, device="cpu")


def test_alloc_layout():
    c = kv4.kv4_alloc(3, 48, 2, 128, device="cpu")
    assert c.shape == (3, 2, 3, 18 * 128) and c.dtype == torch.uint8


def test_heads_describes_strides():
    x = t(6, 5, 64)[:, 1:3]
    at, tok, head, n = struct.unpack("@Pqqi4x", _args.heads(x, "x", torch.bfloat16, CPU, 6, 64))
    assert (at, tok, head, n) == (x.data_ptr(), 320, 64, 2)
    one = t(6, 5, 64)[:1, :1]  # strides of axes of one element count for nothing
    assert struct.unpack("@Pqqi4x", _args.heads(one, "x", torch.bfloat16, CPU, 1, 64))[1:] == (0, 0, 1)


@pytest.mark.parametrize("x", [t(6, 2, 64)[:, :, ::2], t(6, 2, 68)[:, :, :64], t(6, 2, 72)[:, :, 4:68], t(6, 2, 64, dtype=torch.float16),
                               t(6, 64), t(5, 2, 64), t(6, 2, 32), t(6, 0, 64), None])
def test_heads_refuses(x):
    with pytest.raises(ValueError):
        _args.heads(x, "x", torch.bfloat16, CPU, 6, 64)


def test_overlapping_outputs_are_refused():
    ok = [t(6, 2, 64), t(2, 6, 64).transpose(0, 1), t(6, 5, 64)[:, 1:3], t(1, 2, 64), t(6, 1, 64)]
    for x in ok:
        _args.heads(x, "x", torch.bfloat16, CPU, x.shape[0], 64, written=True)
    for x in (t(1, 2, 64).expand(6, 2, 64), t(6, 1, 64).expand(6, 2, 64), torch.as_strided(t(1000), (6, 2, 64), (64, 64, 1)),
              torch.as_strided(t(1000), (6, 2, 64), (120, 64, 1)), torch.as_strided(t(1000), (6, 2, 64), (32, 256, 1))):
        _args.heads(x, "x", torch.bfloat16, CPU, 6, 64)  # read it may be
        with pytest.raises(ValueError):
            _args.heads(x, "x", torch.bfloat16, CPU, 6, 64, written=True)


def test_vector_and_rope_checks():
    i = torch.zeros(6, dtype=torch.int32)
    for bad in (i[:5], i.long(), i.view(2, 3), torch.zeros(12, dtype=torch.int32)[::2], 3):
        with pytest.raises(ValueError):
            _args.vector(bad, "x", torch.int32, 6, CPU)
    f = torch.zeros(32)
    _args.rope_of(i, f, None, t(64), 0.0, True, torch.bfloat16, CPU, 6, 64)
    for bad in (dict(inv_freq=torch.zeros(4)), dict(inv_freq=torch.zeros(36)), dict(inv_freq=torch.zeros(40)), dict(inv_freq=f.double()),
                dict(inv_freq=f.view(4, 8)), dict(positions=i.long()), dict(q_weight=t(32)), dict(q_weight=torch.zeros(64)),
                dict(k_weight=t(72)[1:65]), dict(eps=-1e-6)):
        d = dict(positions=i, inv_freq=f, q_weight=None, k_weight=None, eps=1e-6)
        d.update(bad)
        with pytest.raises(ValueError):
            _args.rope_of(**d, interleaved=False, dtype=torch.bfloat16, index=CPU, tokens=6, dim=64)
